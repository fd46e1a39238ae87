// Choosing a token: temperature, top-k, top-p and min-p over a row of logits, and the inverse of the
// cumulative distribution at a given random number, one launch.
//
//   w_i = exp((x_i - max x) / T)                    T <= 0: the arg max
//   ranked by x, equal values by index:  top-k keeps the first k;  top-p keeps those of them whose
//   predecessors weigh less than p times what top-k kept;  min-p keeps w_i >= min_p.
//   token = the first kept index i, in vocabulary order, with  sum_{j <= i, kept} w_j > u Z
//
// All three filters keep a head of the ranking, so a row needs no sort: the threshold is the value
// K at which the count (top-k) or the weight (top-p) of the values above crosses its target, found by
// histograms over ever smaller ranges of values, plus the number m of values equal to K that are still
// kept (the first m by index).
//
// Weights are integers: exp in 64 bits, scaled by 2^84 and rounded, in two words that are added up apart (2^43, and a
// signed rest).  Their sums are exact, so neither the split over threads and CTAs nor the order of the atomics changes a
// result, and a decision next to a border is the one that 64-bit arithmetic makes, in a long tail of tiny weights too:
// a weight is off by 2^-42 of itself and 2^-85 of the largest.  With one word of 2^44 a tail at 2^-45 of the largest was
// lost altogether, 2^-28 of the whole at V = 128256.  The histogram of top-p takes them in steps of 2^-43, and where a
// border is not clear by what that may be off (few rows) again in steps of 2^-59, so top-p is right to V 2^-60 of the
// whole.  What rounds to zero even so is only ever chosen at u = 0.
//
// A thread-block cluster owns a row: each CTA stages its slice of the row in shared memory (read once
// from HBM) and the passes run there; histograms, maxima and sums meet through distributed shared memory.
//
// Bound: phases.  A row is a chain of passes with barriers of the CTA and the cluster between them, and two CTAs of 512
// threads per SM (three without bins) do not cover one another's waits: warps spend a third of their time at barriers,
// 42 to 53 % of the issue slots are taken, HBM runs at 0.4 to 1.4 TB/s.  Behind that come instructions: a pass costs a
// logit 10 to 60 of them.  One row of 32000 f32 with top-p: 19 us, seven cluster barriers and as many passes of latency.
// 64 rows of 128256 bf16 with mixed filters: 56 us; all with top-p 68 us, of which some 16 us are the weighted histogram
// (shared atomics at 16 cycles a warp each: bank conflicts, not the form of the atomic).  256 rows of 128256 f32
// unfiltered: 114 us where the settings are arrays, and so unknown to the host, else 95 us; 18 % of these flat rows are
// decided by exact sums after all.  What the exact tails cost: 16.6 / 53 / 62.8 / 112 / 93.5 us without them.
// Shared memory counts twice: with 6 KB more a CTA still two fit an SM, but the L1 cache gave way and the loads of a row
// lost 8 % (unfiltered 115 -> 123 us).  Measured and not kept: 256 threads or no staging (unfiltered 92 us, but top-p 80
// to 145 us), 1024 threads (257 us), the estimate while the row streams in (one barrier less, but registers spill),
// always the fine histogram (top-p 68 -> 83 us), both histograms as code of their own (registers).
#include "common.cuh"
#include "capi_internal.h"
#include <math.h>
#include <stddef.h>
#include <type_traits>

namespace arke {

typedef unsigned long long u64;
typedef unsigned __int128 u128;

constexpr int kSmpThreads = 512;
constexpr int kSmpWarps = kSmpThreads / 32;
constexpr int kSmpBins = 2048;
constexpr int kSmpMaxCluster = 8;

struct SampleParams {
  const char* x;
  int64_t ld;
  const float* u;
  const float* t_row;
  const int* k_row;
  const float* p_row;
  const float* m_row;
  float t, p, m;
  int k;
  int64_t* token;
  float* logprob;
  int B, V, slice, staged, stage_at;
};

template <typename T> struct SmpType;
// kGranule: low bits of the fp32 pattern that are the same for every value of the type
template <> struct SmpType<__nv_bfloat16> {
  static constexpr int kGranule = 16;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
};
template <> struct SmpType<__half> {
  static constexpr int kGranule = 13;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
};
template <> struct SmpType<float> {
  static constexpr int kGranule = 0;
  static __device__ __forceinline__ float get(float v) { return v; }
};

// NaN is read as -inf (never chosen), -0 as +0 (they compare equal)
__device__ __forceinline__ float smp_clean(float f) { return fmaxf(f, -INFINITY) + 0.f; }
// unsigned pattern in the order of the values (of a cleaned value)
__device__ __forceinline__ uint32_t smp_key(float f) {
  const int b = __float_as_int(f);
  return (uint32_t)(b ^ ((b >> 31) | 0x80000000));
}
__device__ __forceinline__ float smp_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));   // volatile: stays behind the barriers
  return v;
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const u64 o = __shfl_xor_sync(0xffffffffu, v, d);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v) {   // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += o;
  }
  return v;
}

__device__ __forceinline__ u128 shfl_xor(u128 v, int d) {
  const u64 lo = __shfl_xor_sync(0xffffffffu, (u64)v, d), hi = __shfl_xor_sync(0xffffffffu, (u64)(v >> 64), d);
  return ((u128)hi << 64) | lo;
}
__device__ __forceinline__ u64 shfl_xor(u64 v, int d) { return __shfl_xor_sync(0xffffffffu, v, d); }
__device__ __forceinline__ double real(u128 v) { return (double)(u64)(v >> 64) * 18446744073709551616.0 + (double)(u64)v; }

// f in [0, 1) as the integer m < 2^24 times 2^-e
__device__ __forceinline__ uint32_t as_ratio(float f, int& e) {
  const uint32_t b = __float_as_uint(f), x = b >> 23;
  e = 150 - (x ? (int)x : 1);
  return (b & 0x7fffffu) | (x ? 0x800000u : 0u);
}

constexpr double kSmpOne = 8796093022208.0;    // 2^43: 2^20 of them add up in 64 bits
constexpr int kSmpLow = 41;                    // bits of a weight below that
constexpr double kSmpFine = 65536.0;           // the histogram's steps are finer by this

// sums of a part of a row: weights in two words, and how many equal the threshold
struct Part {
  u64 hi, lo, n;
};
__device__ __forceinline__ Part operator+(Part a, Part b) { return {a.hi + b.hi, a.lo + b.lo, a.n + b.n}; }
__device__ __forceinline__ Part operator-(Part a, Part b) { return {a.hi - b.hi, a.lo - b.lo, a.n - b.n}; }
__device__ __forceinline__ Part lane_of(Part v, int lane) {
  return {__shfl_sync(0xffffffffu, v.hi, lane), __shfl_sync(0xffffffffu, v.lo, lane), __shfl_sync(0xffffffffu, v.n, lane)};
}
template <int N>
__device__ __forceinline__ Part lane_scan(Part v) {      // inclusive, over N lanes
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < N; d <<= 1) {
    const Part o{__shfl_up_sync(0xffffffffu, v.hi, d), __shfl_up_sync(0xffffffffu, v.lo, d), __shfl_up_sync(0xffffffffu, v.n, d)};
    if (lane >= d) v = v + o;
  }
  return v;
}

struct SmpShared {
  double table[16];                         // 2^(j / 16) scaled by 2^43
  u64 warp[kSmpWarps], warp2[kSmpWarps], warp3[kSmpWarps];
  u64 slot[5][kSmpMaxCluster];              // one value from each CTA of the cluster
  u64 res[4];                               // what one CTA found, pushed to all
  u64 sure;                                 // the estimate decided the row
  Part before;                              // what lies before the warp's part that holds the token
  u128 target;                              // the token is the first whose running sum exceeds it
  double log_z;
  int where;                                // that warp, or -1: another CTA's
  alignas(16) uint32_t bin[4][kSmpBins];    // a bin's sum in words of Row::limb bits and what the additions carry
  uint32_t count;                           // values of one bin in this CTA
  // The values of one bin, once the histogram has been read: this CTA's in bin[0] and bin[1], the cluster's in bin[2].
  __device__ __forceinline__ uint32_t* near_key() { return bin[0]; }
  __device__ __forceinline__ u64* near_weight() { return reinterpret_cast<u64*>(bin[1]); }
  __device__ __forceinline__ u64* list() { return reinterpret_cast<u64*>(bin[2]); }
  __device__ __forceinline__ uint32_t* list_key() { return bin[2] + 2 * kSmpThreads; }
};
// the structure lies at a multiple of 128 bytes; 64-bit weights in the bins
static_assert(offsetof(SmpShared, bin) % 16 == 0 && offsetof(SmpShared, target) % 16 == 0 && kSmpBins % 4 == 0);
static_assert(3 * kSmpThreads <= kSmpBins && kSmpWarps * 160 <= 4 * kSmpBins);

template <typename T, int CS>
struct Row {
  const T* src;        // this CTA's slice
  int n, first;        // its length, its first index in the row
  float top;           // the row's maximum
  float base;          // the maximum, or the largest finite value where that is infinite
  float cut;           // values below weigh nothing
  double rate;         // 16 log2(e) / T
  double inv_t;
  SmpShared* s;
  uint32_t rank;
  int limb;            // bits of a histogram word: 32 less what the slice's additions can carry
  bool fine;           // weights go to the histogram in steps of 2^-59, else 2^-43

  // Comparisons take a NaN as it is: it is above nothing and equal to nothing, like the -inf it stands for.
  __device__ __forceinline__ float at(int i) const { return SmpType<T>::get(src[i]); }
  __device__ __forceinline__ uint32_t key(float f) const { return smp_key(smp_clean(f)) >> SmpType<T>::kGranule; }
  __device__ __forceinline__ float value(uint32_t k) const {     // inverse of key()
    const uint32_t full = k << SmpType<T>::kGranule;
    return smp_value(full & 0x80000000u ? full : full | ((1u << SmpType<T>::kGranule) - 1));
  }
  // exp((f - top) / T) * 2^43.  With x = 16 log2(e) (f - top) / T = 16 e + j + r, |r| <= 1/2, it is
  // 2^e * table[j] * 2^(r / 16): twelve 64-bit operations and a 16-entry table whose entries lie in different banks;
  // the Taylor polynomial of degree 5 leaves (ln 2 / 32)^6 / 6! = 2^-42.7.  f == top gives 2^43 exactly.
  // Without branches, so that several elements are in flight: what `cut` drops is computed and thrown away.
  __device__ __forceinline__ double scaled(float f) const {
    const double x = ((double)fminf(f, base) - (double)base) * rate;
    const double magic = 6755399441055744.0;                     // 1.5 * 2^52: the sum's low bits are round(x)
    const double xm = x + magic;
    const int n = __double2loint(xm);
    const double r = x - (xm - magic);
    constexpr double c = 0.043321698784996581838;                // ln 2 / 16
    double y = fma(r, c * c * c * c * c / 120, c * c * c * c / 24);
    y = fma(r, y, c * c * c / 6);
    y = fma(r, y, c * c / 2);
    y = fma(r, y, c);
    const double tj = s->table[n & 15];
    y = fma(r * y, tj, tj);
    y = __hiloint2double(__double2hiint(y) + ((n >> 4) << 20), __double2loint(y));
    return f >= cut ? y : 0.0;
  }
  // that times 2^41, rounded, as hi 2^41 + lo with a signed lo: the rounded value and what is left of it, which is exact.
  // Added to hi and lo as the bits of a double that has them in its low end, kHi and kLo above what they are.
  static constexpr u64 kHi = 0x4330000000000000ull, kLo = 0x4338000000000000ull;     // 2^52, 1.5 * 2^52
  static __device__ __forceinline__ void add_raw(double y, u64& hi, u64& lo) {
    const double big = 4503599627370496.0, magic = 6755399441055744.0;
    const double up = y + big;
    hi += (u64)__double_as_longlong(up);
    lo += (u64)__double_as_longlong(fma(y - (up - big), (double)(1ull << kSmpLow), magic));
  }
  static __device__ __forceinline__ u128 join(u64 hi, u64 lo) { return ((u128)hi << kSmpLow) + (u128)(__int128)(long long)lo; }
  __device__ __forceinline__ u128 weight(float f) const {
    u64 hi = 0, lo = 0;
    add_raw(scaled(f), hi, lo);
    return join(hi - kHi, lo - kLo);
  }
  // in the histogram's steps
  __device__ __forceinline__ u64 binned(float f) const {
    return __double2ull_rn(scaled(f) * (fine ? kSmpFine : 1.0));
  }
  // coarse bin of a value, 0 = the highest: 1/64 of a logit each, the last takes the rest (and NaN)
  __device__ __forceinline__ int coarse(float f) const {
    return (int)__float2uint_rz(fminf((base - f) * 64.f, (float)(kSmpBins - 1)));
  }

  // the CTA's value (every thread has it) to slot[which][rank] of every CTA, one thread for each
  __device__ __forceinline__ void push(int which, u64 v) const {
    if (threadIdx.x < CS) st_cluster_u64(mapa_cluster(smem_u32(&s->slot[which][rank]), threadIdx.x), v);
  }
};

// Inclusive scan over the CTA of one value per thread: the sum up to this thread, and of all.
__device__ __forceinline__ u64 block_scan(u64 v, u64* part, u64& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  u64 inc = warp_scan(v);
  __syncthreads();
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kSmpWarps; ++w) {
    const u64 x = part[w];
    if (w < warp) inc += x;
    total += x;
  }
  return inc;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ u64 bits(double v) { return (u64)__double_as_longlong(v); }
__device__ __forceinline__ double real(u64 v) { return __longlong_as_double((long long)v); }

// Where neither top-k nor top-p asks for a threshold, all that is decided is where u Z falls among the running sums,
// and single precision mostly can tell: a weight costs six instructions instead of thirty.  The sums carry a bound of
// their error: ex2 is good to 2^-22, eight weights are added in a tree of depth three before they go to 64 bits, and
// the exponent t, three roundings of 2^-24, adds ln 2 * 3 * |t| * 2^-24 of the weight, for which sum w |t| is kept too:
//   |error of any running sum| <= E = 2^-24 (7 Z + 2.1 sum w |t|).
// The hundredth that is added to E covers what `least` leaves out, 2^20 weights of 2^-48 at most; so a first token is
// not sure either while u Z lies within that of zero.
// A token whose running sums lie further than 2 E from u Z on both sides is the one that exact sums would choose;
// else the row is decided by those.  Returns whether it is done.  A function of its own, so that what follows in the kernel
// does not cost its loops registers (256 x 128256 f32 with min-p: 84 -> 80 us).
template <typename T, int CS>
__device__ __noinline__ bool estimate(Row<T, CS> r, const SampleParams& p, int row, float least, float u) {
  SmpShared& s = *r.s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float rate = (float)(r.inv_t * 1.4426950408889634), base = r.base;
  if (!(rate <= 3.0e38f)) return false;                  // a temperature too small for single precision
  auto weight = [&](float f, float& t) {
    t = (fminf(f, base) - base) * rate;
    return f >= least ? ex2_approx(t) : 0.f;             // false for NaN; t of a dropped value only meets weight 0
  };
  const int part = (r.n + kSmpWarps * 32 - 1) / (kSmpWarps * 32) * 32;
  const int i0 = min(warp * part, r.n), i1 = min(i0 + part, r.n);
  double z = 0.0, dev = 0.0;
  int i = i0 + lane;
  for (; i + 7 * 32 < i1; i += 8 * 32) {
    float w[8], d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float t;
      w[e] = weight(r.at(i + e * 32), t);
      d[e] = w[e] * fmaxf(t, -200.f);                    // finite times zero
    }
    z += (double)(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
    dev += (double)(((d[0] + d[1]) + (d[2] + d[3])) + ((d[4] + d[5]) + (d[6] + d[7])));
  }
  for (; i < i1; i += 32) {
    float t;
    const float w = weight(r.at(i), t);
    z += (double)w;
    dev += (double)(w * fmaxf(t, -200.f));
  }
  z = warp_sum(z);
  dev = warp_sum(dev);
  if (lane == 0) { s.warp[warp] = bits(z); s.warp2[warp] = bits(dev); }
  __syncthreads();
  z = dev = 0.0;
#pragma unroll
  for (int w = 0; w < kSmpWarps; ++w) { z += real(s.warp[w]); dev += real(s.warp2[w]); }
  r.push(3, bits(z));
  r.push(4, bits(dev));
  cluster_sync_all();
  double total = 0.0, mine = 0.0;
  dev = 0.0;
#pragma unroll
  for (uint32_t c = 0; c < CS; ++c) {
    if (c == r.rank) mine = total;
    total += real(s.slot[3][c]);
    dev -= real(s.slot[4][c]);
  }
  const double bound = 1.01 * 5.9604644775390625e-8 * (7.0 * total + 2.1 * dev), target = (double)u * total;
  int where = -1;
  for (int w = 0; w < kSmpWarps; ++w) {
    const double a = real(s.warp[w]);
    if (mine <= target && target < mine + a) { where = w; break; }
    mine += a;
  }
  if (where >= 0) {                                      // this CTA's: its part once more, a few neighbours a thread
    const int j0 = min(where * part, r.n), j1 = min(j0 + part, r.n);
    const int per = (part + kSmpThreads - 1) / kSmpThreads;
    const int e0 = min(j0 + tid * per, j1), e1 = min(e0 + per, j1);
    float t;
    double sum = 0.0;
    for (int e = e0; e < e1; ++e) sum += (double)weight(r.at(e), t);
    double inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += v;
    }
    __syncthreads();
    if (lane == 31) s.warp2[warp] = bits(inc);
    __syncthreads();
    for (int w = 0; w < warp; ++w) inc += real(s.warp2[w]);
    mine += inc - sum;
    if (mine <= target && target < mine + sum) {
      for (int e = e0; e < e1; ++e) {
        const float f = r.at(e);
        const double next = mine + (double)weight(f, t);
        if (target < next) {
          if (next - target > 2.0 * bound && target - mine > 2.0 * bound) {
            p.token[row] = r.first + e;
            if (p.logprob) p.logprob[row] = (float)((f == r.top ? 0.0 : ((double)f - (double)r.top) * r.inv_t) - log(total));
#pragma unroll
            for (uint32_t c = 0; c < CS; ++c) st_cluster_u64(mapa_cluster(smem_u32(&s.sure), c), 1ull);
          }
          break;
        }
        mine = next;
      }
    }
  }
  cluster_sync_all();
  return s.sure != 0;
}

// Counts fit 64 bits, sums of weights do not.
template <bool WEIGHT> using Sum = std::conditional_t<WEIGHT, u128, u64>;

// What is looked for: a sum of at least `target`, or, where that is 0, of at least `share` of (all - surplus).
template <bool WEIGHT>
struct Goal {
  Sum<WEIGHT> target;
  float share;         // in [0, 1)
  Sum<WEIGHT> surplus;
};

// Looks for the bin in which the sum from bin 0 on reaches the goal: its index, how much of the goal the bins before
// it leave to it, and (counts) what it holds, to res[] of every CTA.  The bins of all CTAs are added up first.
template <bool WEIGHT, typename T, int CS>
__device__ __forceinline__ void find_bin(Row<T, CS>& r, const Goal<WEIGHT>& goal) {
  SmpShared& s = *r.s;
  const int tid = threadIdx.x, limb = r.limb;
  constexpr int nb = kSmpBins / CS, per = (nb + kSmpThreads - 1) / kSmpThreads;
  cluster_sync_all();                                   // every CTA's bins are complete
  auto read = [&](int e, u64& lo, u64& hi) {            // this thread's e-th bin is lo + 2^(2 limb) hi
    const uint32_t from = smem_u32(&s.bin[0][r.rank * nb + tid * per + e]);
    constexpr int W = WEIGHT ? 4 : 1;
    uint32_t l[CS][W];                                  // all loads in flight before the first is used
#pragma unroll
    for (uint32_t c = 0; c < CS; ++c)
#pragma unroll
      for (int w = 0; w < W; ++w) l[c][w] = w == 3 && !r.fine ? 0 : ld_cluster_u32(mapa_cluster(from + w * kSmpBins * 4, c));
    lo = hi = 0;
#pragma unroll
    for (int c = 0; c < CS; ++c) {
      lo += l[c][0];
      if constexpr (WEIGHT) {
        lo += (u64)l[c][1] << limb;
        hi += l[c][2] + ((u64)l[c][3] << limb);         // l[c][3] only where the steps are fine
      }
    }
  };
  u64 mine_lo = 0, mine_hi = 0;
#pragma unroll
  for (int e = 0; e < per; ++e) {
    if (tid * per + e >= nb) break;
    u64 lo, hi;
    read(e, lo, hi);
    mine_lo += lo;
    mine_hi += hi;
  }
  // in steps of 2^-43 a row's sum fits one word
  const bool wide = WEIGHT && r.fine;
  if (WEIGHT && !wide) { mine_lo += mine_hi << (2 * limb); mine_hi = 0; }
  auto sum = [&](u64 low, u64 high) -> Sum<WEIGHT> {
    if constexpr (WEIGHT) return ((u128)high << (2 * limb)) + low;
    else return low;
  };
  u64 total_lo, total_hi = 0, end_lo = block_scan(mine_lo, s.warp, total_lo), end_hi = 0;
  if (wide) end_hi = block_scan(mine_hi, s.warp2, total_hi);
  r.push(0, total_lo);
  if (wide) r.push(1, total_hi);
  cluster_sync_all();
  Sum<WEIGHT> target = goal.target;
  u64 all_lo = 0, all_hi = 0;
  for (uint32_t c = 0; c < CS; ++c) {
    const u64 v = s.slot[0][c], w = wide ? s.slot[1][c] : 0;
    if (c < r.rank) { end_lo += v; end_hi += w; }
    all_lo += v;
    all_hi += w;
  }
  if constexpr (WEIGHT) {
    if (target == 0) {
      int shift;
      const u128 want = (u128)(sum(all_lo, all_hi) - goal.surplus) * as_ratio(goal.share, shift);     // 2^79 * 2^24 at most
      target = shift >= 128 ? want != 0 : (Sum<WEIGHT>)(want >> shift) + ((want & (((u128)1 << shift) - 1)) != 0);
      if (target == 0) target = 1;
    }
  }
  const Sum<WEIGHT> end = sum(end_lo, end_hi);
  Sum<WEIGHT> begin = sum(end_lo - mine_lo, end_hi - mine_hi);
  if (begin < target && target <= end) {
    int e = 0;
    Sum<WEIGHT> v = sum(mine_lo, mine_hi);
    if constexpr (per > 1) {                            // one thread's: its bins once more
      for (;; ++e) {
        u64 lo, hi;
        read(e, lo, hi);
        v = sum(lo, hi);
        if (target <= begin + v) break;
        begin += v;
      }
    }
    const Sum<WEIGHT> rest = target - begin;
    const u64 found[3] = {(u64)(r.rank * nb + tid * per + e), (u64)rest, WEIGHT ? (u64)((u128)rest >> 64) : (u64)v};
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
      for (uint32_t c = 0; c < CS; ++c) st_cluster_u64(mapa_cluster(smem_u32(&s.res[i]), c), found[i]);
  }
  cluster_sync_all();
}
template <bool WEIGHT>
__device__ __forceinline__ Sum<WEIGHT> found_rest(const SmpShared& s) {
  if constexpr (WEIGHT) return ((u128)s.res[2] << 64) | s.res[1];
  else return s.res[1];
}

template <bool WEIGHT>
__device__ __forceinline__ void clear_bins(SmpShared& s, bool fine) {
  const int words = !WEIGHT ? 1 : fine ? 4 : 3;
  for (int j = threadIdx.x; j < words * kSmpBins / 4; j += kSmpThreads) reinterpret_cast<uint4*>(s.bin)[j] = make_uint4(0, 0, 0, 0);
  __syncthreads();
}
// Adds without reading back: an atomic whose result nobody waits for costs a slot, not a round trip.
template <bool WEIGHT>
__device__ __forceinline__ void add_bin(SmpShared& s, int limb, int bin, u64 w) {
  if constexpr (!WEIGHT) {
    atomicAdd(&s.bin[0][bin], 1u);
  } else {
    const uint32_t mask = (1u << limb) - 1, low = (uint32_t)w, high = (uint32_t)(w >> 32);
    const uint32_t upper = limb >= 16 ? high >> (2 * limb - 32) : __funnelshift_r(low, high, 2 * limb);       // of 2^59 at most
    atomicAdd(&s.bin[0][bin], low & mask);
    atomicAdd(&s.bin[1][bin], __funnelshift_r(low, high, limb) & mask);
    if (upper) {                                         // slices of 2^14: 2^-7 of the largest weight and more, or 2^-23
      atomicAdd(&s.bin[2][bin], upper & mask);
      if (upper >> limb) atomicAdd(&s.bin[3][bin], upper >> limb);
    }
  }
}

// The largest value (key K) with (count or weight of the values >= it) >= the goal, over the values that are not
// below `least`; how much of the goal the values above it leave to those equal to it, and (counts) how many these are.
template <bool WEIGHT, typename T, int CS>
__device__ __forceinline__ void find_threshold(Row<T, CS>& r, const Goal<WEIGHT>& goal, float least, uint32_t& K, Sum<WEIGHT>& rest, u64& equals) {
  SmpShared& s = *r.s;
  const int tid = threadIdx.x;
  clear_bins<WEIGHT>(s, r.fine);
#pragma unroll 4
  for (int i = tid; i < r.n; i += kSmpThreads) {
    const float f = r.at(i);
    if (f < least) continue;
    add_bin<WEIGHT>(s, r.limb, r.coarse(f), WEIGHT ? r.binned(f) : 1);
  }
  find_bin<WEIGHT>(r, goal);
  const int coarse = (int)s.res[0];
  // keys that the coarse bin may hold, a little more on both sides than its rounding can reach
  const double step = 1.0 / 64, top = (double)r.top;
  const double slack = 1e-6 * (fabs(top) + (coarse + 1) * step);
  uint32_t khi = coarse == 0 ? r.key(r.top) : r.key(fminf((float)(top - coarse * step + slack), r.top));
  uint32_t klo = coarse == kSmpBins - 1 ? 0u : r.key((float)(top - (coarse + 1) * step - slack));
  if (r.top == INFINITY) klo = 0u;                       // bins of infinite width
  if (klo < khi) {
    // A bin of few values is resolved in one step: every CTA gets all of them and adds up, for each of its own, what
    // lies above it and what equals it.
    uint32_t* const near_key = s.near_key();
    u64* const near_weight = s.near_weight();
    if (tid == 0) s.count = 0;
    __syncthreads();
    for (int i0 = tid; i0 < r.n; i0 += 4 * kSmpThreads) {
      float f[4];
      bool in[4], any = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e * kSmpThreads;
        f[e] = i < r.n ? r.at(i) : 0.f;
        in[e] = i < r.n && r.coarse(f[e]) == coarse && !(f[e] < least);
        any |= in[e];
      }
      if (!any) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!in[e]) continue;
        const u64 w = WEIGHT ? r.binned(f[e]) : 1;
        if (!w) continue;
        const uint32_t at = atomicAdd(&s.count, 1u);
        if (at < kSmpThreads) {
          near_key[at] = r.key(f[e]);
          near_weight[at] = w;
        }
      }
    }
    __syncthreads();
    const uint32_t own = s.count;
    r.push(0, own);
    cluster_sync_all();
    uint32_t n = 0, first = 0;
#pragma unroll
    for (uint32_t c = 0; c < CS; ++c) {
      const uint32_t m = (uint32_t)s.slot[0][c];
      if (c < r.rank) first += m;
      n += m;
    }
    if (n <= kSmpThreads) {
      if (tid < (int)own) {
        const uint32_t k = near_key[tid];
        const u64 w = near_weight[tid];
#pragma unroll
        for (uint32_t c = 0; c < CS; ++c) {
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_cluster(smem_u32(&s.list_key()[first + tid]), c)), "r"(k) : "memory");
          st_cluster_u64(mapa_cluster(smem_u32(&s.list()[first + tid]), c), w);
        }
      }
      const Sum<WEIGHT> left = found_rest<WEIGHT>(s);
      cluster_sync_all();
      // eight lanes to each of this CTA's own values
      for (uint32_t e0 = 0; e0 < own; e0 += kSmpThreads / 8) {
        const uint32_t e = e0 + tid / 8, k = s.list_key()[first + min(e, own - 1)];
        Sum<WEIGHT> more = 0, same = 0;
#pragma unroll 4
        for (uint32_t i = tid & 7; i < n; i += 8) {
          const u64 w = s.list()[i];
          const uint32_t ki = s.list_key()[i];
          more += ki > k ? w : 0;
          same += ki == k ? w : 0;
        }
#pragma unroll
        for (int d = 4; d; d >>= 1) {
          more += shfl_xor(more, d);
          same += shfl_xor(same, d);
        }
        if (more < left && left <= more + same && (tid & 7) == 0) {   // equal values all write the same
          const u64 found[3] = {k, (u64)(left - more), WEIGHT ? (u64)((u128)(left - more) >> 64) : (u64)same};
#pragma unroll
          for (int i = 0; i < 3; ++i)
#pragma unroll
            for (uint32_t c = 0; c < CS; ++c) st_cluster_u64(mapa_cluster(smem_u32(&s.res[i]), c), found[i]);
        }
      }
      cluster_sync_all();
      K = (uint32_t)s.res[0];
      rest = found_rest<WEIGHT>(s);
      equals = s.res[2];
      __syncthreads();
      return;
    }
    cluster_sync_all();                                  // the list is read no more: the bins are free again
  }
  while (klo < khi) {
    const uint32_t span = khi - klo;
    const int bits = 32 - __clz(span), shift = bits > 11 ? bits - 11 : 0;
    const Goal<WEIGHT> left{found_rest<WEIGHT>(s), 0.f, 0};
    clear_bins<WEIGHT>(s, r.fine);
#pragma unroll 4
    for (int i = tid; i < r.n; i += kSmpThreads) {
      const float f = r.at(i);
      if (r.coarse(f) != coarse || f < least) continue;
      const uint32_t k = r.key(f);
      if (k < klo || k > khi) continue;
      const u64 w = WEIGHT ? r.binned(f) : 1;
      if (w) add_bin<WEIGHT>(s, r.limb, (int)((khi - k) >> shift), w);
    }
    find_bin<WEIGHT>(r, left);
    const int bin = (int)s.res[0];
    khi -= (uint32_t)bin << shift;
    const uint32_t low = khi - ((1u << shift) - 1);
    klo = low > klo && low <= khi ? low : klo;
    if (shift == 0) klo = khi;
  }
  K = khi;
  rest = found_rest<WEIGHT>(s);
  equals = s.res[2];
  __syncthreads();
}

// the least n with n w >= rest, for a rest of up to 2^20 w
__device__ __forceinline__ u64 how_many(u128 rest, u64 w) {
  if (w == 0 || rest <= w) return 1;
  u64 n = (u64)(real(rest) / (double)w);
  while (n > 1 && (u128)(n - 1) * w >= rest) --n;
  while ((u128)n * w < rest) ++n;
  return n;
}

// Top-p among the values that are not below `least`, of which the last `surplus` equal to it stay out: the threshold K
// and how many of its equals stay in.  In steps of 2^-43 every weight is off by half a step, the difference of a running
// sum and p Z so by less than V of them: a border further away than that is where it is in 64 bits too, else the steps
// are made finer.
template <typename T, int CS>
__device__ __forceinline__ void find_top_p(Row<T, CS>& r, float p, float least, u64 surplus, int V, uint32_t& K, u64& allowed) {
  for (r.fine = false;; r.fine = true) {
    u128 rest;
    u64 unused;
    find_threshold<true>(r, Goal<true>{0, p, surplus ? (u128)surplus * r.binned(least) : 0}, least, K, rest, unused);
    const float f = r.value(K);
    const u64 w = r.binned(f), margin = (u64)V + 2;
    allowed = how_many(rest, w);
    if (r.fine) return;
    const bool first = allowed == 1 && f == r.top;       // stays in whatever its predecessors, none, weigh
    const u128 over = (u128)allowed * w - rest;          // w = 0: wraps, but then nothing is clear
    if (w > margin && over > margin && (first || w - (u64)over > margin)) return;
  }
}

// FILTERS: some row may have a top-k or top-p
template <typename T, int CS, bool FILTERS>
__global__ void __launch_bounds__(kSmpThreads, FILTERS ? 2 : 3) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  SmpShared& s = *reinterpret_cast<SmpShared*>(smem);
  T* stage = reinterpret_cast<T*>(smem + p.stage_at);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  Row<T, CS> r;
  r.rank = CS == 1 ? 0 : cluster_ctarank();
  r.s = &s;
  r.fine = false;
  const int row = blockIdx.x / CS;
  r.first = (int)r.rank * p.slice;
  r.n = max(0, min(p.slice, p.V - r.first));
  r.limb = __clz(p.slice - 1);                           // slice <= 2^(32 - limb); 15 bits at V = 2^20
  const T* src = reinterpret_cast<const T*>(p.x) + (int64_t)row * p.ld + r.first;
  r.src = p.staged ? stage : src;
  if (!ARKE_CHK(row, row, p.B)) return;                  // every setting and output of the row; the same for the whole cluster
  const float t = p.t_row ? p.t_row[row] : p.t, pp = p.p_row ? p.p_row[row] : p.p;
  const float r_min_p = fminf(p.m_row ? p.m_row[row] : p.m, 1.f);
  const int k = p.k_row ? p.k_row[row] : p.k;
  const float u_row = p.u[row];
  if (tid == 0) s.sure = 0;
  if constexpr (CS > 1) cluster_arrive_relaxed();        // every CTA has begun before the first push

  // ---- the slice and its maximum (a NaN never is one)
  float best = -INFINITY;
  constexpr int VEC = 16 / sizeof(T);
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const int nv = r.n / VEC;
    done = nv * VEC;
#pragma unroll 8
    for (int j = tid; j < nv; j += kSmpThreads) {
      const int64_t e = (int64_t)r.first + j * VEC;
      if (!ARKE_CHK(e, e + VEC - 1, p.V)) continue;
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(src) + j);
      if (p.staged) reinterpret_cast<uint4*>(stage)[j] = q;
      const T* v = reinterpret_cast<const T*>(&q);
#pragma unroll
      for (int i = 0; i < VEC; ++i) best = fmaxf(best, SmpType<T>::get(v[i]));
    }
  }
#pragma unroll 8
  for (int i = done + tid; i < r.n; i += kSmpThreads) {
    if (!ARKE_CHK(r.first + i, r.first + i, p.V)) continue;
    const T v = src[i];
    if (p.staged) stage[i] = v;
    best = fmaxf(best, SmpType<T>::get(v));
  }
  u64 top = __reduce_max_sync(0xffffffffu, smp_key(smp_clean(best)));
  if (lane == 0) s.warp[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSmpWarps; ++w) top = s.warp[w] > top ? s.warp[w] : top;
  if constexpr (CS > 1) cluster_wait();
  r.push(0, top);
  cluster_sync_all();
  top = 0;
#pragma unroll
  for (uint32_t c = 0; c < CS; ++c) top = s.slot[0][c] > top ? s.slot[0][c] : top;
  r.top = smp_value((uint32_t)top);

  const bool none = r.top == -INFINITY;
  if (none || !(t > 0.f)) {                              // the same for every CTA of the cluster
    // the lowest index of the maximum, as the maximum of its complement
    u64 at = 0;
    if (!none)
      for (int i = tid; i < r.n; i += kSmpThreads)
        if (r.at(i) == r.top) { at = (uint32_t)~(uint32_t)(r.first + i); break; }
    at = warp_max(at);
    __syncthreads();
    if (lane == 0) s.warp[warp] = at;
    __syncthreads();
    for (int w = 0; w < kSmpWarps; ++w) at = s.warp[w] > at ? s.warp[w] : at;
    r.push(1, at);
    cluster_sync_all();
    if (r.rank == 0 && tid == 0) {
      for (uint32_t c = 0; c < CS; ++c) at = s.slot[1][c] > at ? s.slot[1][c] : at;
      p.token[row] = none ? -1 : (int64_t)(~(uint32_t)at);
      if (p.logprob) p.logprob[row] = none ? -INFINITY : 0.f;
    }
    return;
  }
  r.inv_t = 1.0 / (double)t;
  r.rate = r.inv_t * 23.083120654223415;                 // 16 log2(e)
  // below max - 85.5 ln(2) T a weight rounds to zero
  r.base = fminf(r.top, 3.402823466e38f);
  r.cut = fmaxf((float)((double)r.top - 59.3 * (double)t), -3.402823466e38f);
  if (tid < 16) s.table[tid] = exp2(tid / 16.0) * kSmpOne;
  __syncthreads();

  const float u = u_row > 0.f ? u_row : 0.f;
  // min-p as a limit of the logits: the least float that is not below max + T ln(min_p), less what the exponential of
  // 64 bits rounds up to min_p (2^-54, for min_p = 1 at temperatures that leave nothing of the differences)
  const float floor = r_min_p > 0.f && r.top < INFINITY
                          ? __double2float_ru((double)r.top + (double)t * (log((double)r_min_p) - 5.551115123125783e-17)) : -INFINITY;
  if (!FILTERS || (!(k > 0 && k < p.V) && !(pp < 1.f))) {
    const float cut = fmaxf((float)((double)r.top - 33.3 * (double)t), -3.402823466e38f);      // 2^-48 of the largest
    if (estimate(r, p, row, fmaxf(floor, cut), u)) return;
  }

  // ---- the value that still stays in, and how many of its equals
  uint32_t K = 0;
  u64 allowed = ~0ull;
  if (FILTERS && k > 0 && k < p.V) {
    u64 equals;
    find_threshold<false>(r, Goal<false>{(u64)k, 0.f, 0}, -INFINITY, K, allowed, equals);
    if (pp < 1.f) {
      uint32_t Kp;
      u64 m;
      find_top_p(r, fmaxf(pp, 0.f), r.value(K), equals - allowed, p.V, Kp, m);
      if (Kp != K || m < allowed) allowed = m;
      K = Kp;
    }
  } else if (FILTERS && pp < 1.f) {
    find_top_p(r, fmaxf(pp, 0.f), -INFINITY, 0, p.V, K, allowed);
  }

  // ---- sums of what stays in, in the order of the vocabulary: a contiguous part for each warp
  r.cut = fmaxf(r.cut, floor);
  const bool filtered = FILTERS && allowed != ~0ull;
  const float fk = filtered ? r.value(K) : -INFINITY;    // above it all stay in, of its equals the first `allowed`
  const u128 w_eq = filtered ? r.weight(fk) : 0;
  const int part = (r.n + kSmpWarps * 32 - 1) / (kSmpWarps * 32) * 32;
  const int i0 = min(warp * part, r.n), i1 = min(i0 + part, r.n);
  u64 hi = 0, lo = 0;
  uint32_t eq = 0;
  if (!filtered) {
#pragma unroll 8
    for (int i = i0 + lane; i < i1; i += 32) r.add_raw(r.scaled(r.at(i)), hi, lo);
    const u64 added = i1 > i0 + lane ? (i1 - i0 - lane + 31) / 32 : 0;
    hi -= added * r.kHi;
    lo -= added * r.kLo;
  } else {
    // few stay in: they are queued until there is one for every lane
    float* const queue = reinterpret_cast<float*>(s.bin) + warp * 160;
    int n = 0;
    for (int i = i0; i < i1; i += 4 * 32) {
      float f[4];
      unsigned in[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = i + e * 32 + lane;
        f[e] = j < i1 ? r.at(j) : -INFINITY;
        eq += f[e] == fk && j < i1;
        in[e] = __ballot_sync(0xffffffffu, f[e] > fk);
      }
      if ((in[0] | in[1] | in[2] | in[3]) == 0) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (f[e] > fk) queue[n + __popc(in[e] & ((1u << lane) - 1))] = f[e];
        n += __popc(in[e]);
      }
      __syncwarp();
      while (n >= 32) {                                  // from the end, so that nothing has to move
        n -= 32;
        r.add_raw(r.scaled(queue[n + lane]), hi, lo);
        hi -= r.kHi;
        lo -= r.kLo;
      }
      __syncwarp();
    }
    if (lane < n) {
      r.add_raw(r.scaled(queue[lane]), hi, lo);
      hi -= r.kHi;
      lo -= r.kLo;
    }
  }
  hi = warp_sum(hi);
  lo = warp_sum(lo);
  eq = __reduce_add_sync(0xffffffffu, eq);
  __syncthreads();
  if (lane == 0) { s.warp[warp] = hi; s.warp2[warp] = eq; s.warp3[warp] = lo; }
  __syncthreads();
  // weight of a part, of its values equal to K the first `allowed`
  auto weigh = [&](Part v) { return r.join(v.hi, v.lo) + (v.n < allowed ? v.n : allowed) * w_eq; };
  // One warp for all: lane w has warp w's part, lane c CTA c's.
  Part in_warp{0, 0, 0}, up_to_warp, in_cta;
  if (warp == 0) {
    if (lane < kSmpWarps) in_warp = {s.warp[lane], s.warp3[lane], s.warp2[lane]};
    up_to_warp = lane_scan<kSmpWarps>(in_warp);
    in_cta = lane_of(up_to_warp, kSmpWarps - 1);
    r.push(1, in_cta.hi);
    r.push(2, in_cta.n);
    r.push(3, in_cta.lo);
  }
  cluster_sync_all();
  if (warp == 0) {
    const Part up_to_cta = lane_scan<CS>(lane < CS ? Part{s.slot[1][lane], s.slot[3][lane], s.slot[2][lane]} : Part{0, 0, 0});
    const u128 z = weigh(lane_of(up_to_cta, CS - 1));
    const Part before_cta = lane_of(up_to_cta, r.rank) - in_cta;
    u128 target = z - 1;
    if (u < 1.f) {
      int shift;
      const u128 scaled = z * as_ratio(u, shift);        // 2^104 * 2^24 at most
      target = shift >= 128 ? 0 : scaled >> shift;
    }
    const Part to = before_cta + up_to_warp, from = to - in_warp;
    const bool here = lane < kSmpWarps && weigh(from) <= target && target < weigh(to);
    if (here) s.before = from;
    const unsigned which = __ballot_sync(0xffffffffu, here);
    if (lane == 0) {
      s.target = target;
      s.log_z = log(real(z) / (kSmpOne * (double)(1ull << kSmpLow)));
      s.where = __ffs(which) - 1;
    }
  }
  __syncthreads();
  auto choose = [&](int i, float f) {
    p.token[row] = r.first + i;
    if (p.logprob) p.logprob[row] = (float)((f == r.top ? 0.0 : ((double)f - (double)r.top) * r.inv_t) - s.log_z);
  };
  if (u == 0.f) {
    // The first token that is kept and whose weight is not zero in 64 bits: below e^-745.13 it is.  Its index as the
    // maximum of the complement.
    u64 at = 0;
    for (int i = tid; i < r.n; i += kSmpThreads) {
      const float f = r.at(i);
      const double e = f == r.top ? 0.0 : ((double)f - (double)r.top) * r.inv_t;
      if (f >= fk && f >= floor && e > -745.13) { at = (uint32_t)~(uint32_t)(r.first + i); break; }
    }
    at = warp_max(at);
    __syncthreads();
    if (lane == 0) s.warp[warp] = at;
    __syncthreads();
    for (int w = 0; w < kSmpWarps; ++w) at = s.warp[w] > at ? s.warp[w] : at;
    r.push(0, at);
    cluster_sync_all();
    for (uint32_t c = 0; c < CS; ++c) at = s.slot[0][c] > at ? s.slot[0][c] : at;
    const int i = (int)~(uint32_t)at - r.first;
    if (tid == 0 && i >= 0 && i < r.n) choose(i, r.at(i));
    return;
  }
  const int where = s.where;
  if (where < 0) return;                                 // another CTA's
  const u128 target = s.target;
  // ---- that part once more, spread over the CTA: each thread a few neighbours
  const int j0 = min(where * part, r.n), j1 = min(j0 + part, r.n);
  const int per = (part + kSmpThreads - 1) / kSmpThreads;
  const int e0 = min(j0 + tid * per, j1), e1 = min(e0 + per, j1);
  hi = lo = eq = 0;
  for (int i = e0; i < e1; ++i) {
    const float f = r.at(i);
    if (f == fk) ++eq;
    if (f > fk) {
      r.add_raw(r.scaled(f), hi, lo);
      hi -= r.kHi;
      lo -= r.kLo;
    }
  }
  u64 unused;
  const u64 hi_end = block_scan(hi, s.warp, unused), lo_end = block_scan(lo, s.warp3, unused), eq_end = block_scan(eq, s.warp2, unused);
  Part mine = s.before + Part{hi_end - hi, lo_end - lo, eq_end - eq};
  if (weigh(mine) <= target && target < weigh(mine + Part{hi, lo, eq})) {
    for (int i = e0; i < e1; ++i) {
      const float f = r.at(i);
      if (f == fk) ++mine.n;
      if (f > fk) {
        r.add_raw(r.scaled(f), mine.hi, mine.lo);
        mine.hi -= r.kHi;
        mine.lo -= r.kLo;
      }
      if (weigh(mine) > target) {
        choose(i, f);
        break;
      }
    }
  }
}

constexpr int kSmpMaxSmem = 200 * 1024;

template <typename T, int CS, bool FILTERS>
static int launch_sample_cluster(SampleParams& p, cudaStream_t st) {
  p.slice = ((p.V + CS - 1) / CS + 31) / 32 * 32;
  const int64_t bytes = (int64_t)p.slice * sizeof(T);
  p.stage_at = (int)((FILTERS ? sizeof(SmpShared) : offsetof(SmpShared, bin)) + 127) / 128 * 128;
  p.staged = bytes <= kSmpMaxSmem - p.stage_at;
  const int smem = p.stage_at + (p.staged ? (int)bytes : 0);
  auto kern = sample_kernel<T, CS, FILTERS>;
  cudaError_t e = ensure_dynamic_smem(kern, kSmpMaxSmem);
  if (e != cudaSuccess) return set_cuda_error("sample_tokens shared memory", e);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((int64_t)p.B * CS));
  cfg.blockDim = dim3(kSmpThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CS;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, p);
  return e == cudaSuccess ? ARKE_OK : set_cuda_error("sample_tokens launch", e);
}

// Without top-k and top-p for any row, the kernel that has neither fits an SM three times instead of twice: 40 registers,
// no bins.  Worth it from two CTAs an SM on (256 rows of 128256 f32: 114 -> 95 us; 512 of 50257 f16: 64 -> 55 us), not below (one row of 32000: 5.3 and 5.4 us) nor where a slice is not staged (16 of 2^20: 37 and 39 us).
template <typename T, int CS>
static int launch_sample_filters(SampleParams& p, cudaStream_t st) {
  const bool none = !p.k_row && !p.p_row && p.k == 0 && !(p.p < 1.f);
  const int64_t slice = ((int64_t)p.V + CS - 1) / CS * (int64_t)sizeof(T);
  if (none && (int64_t)p.B * CS > 2 * sm_count() && slice <= 72 * 1024) return launch_sample_cluster<T, CS, false>(p, st);
  return launch_sample_cluster<T, CS, true>(p, st);
}

template <typename T>
static int launch_sample(SampleParams& p, cudaStream_t st) {
  // CTAs per row: enough to hold the row's slices in 72 KB each (two CTAs to an SM), and more while
  // there are SMs without a row.
  constexpr int kStage = 72 * 1024;
  int c = 1;
  while (c < kSmpMaxCluster && (((int64_t)p.V * sizeof(T) + c - 1) / c > kStage || (int64_t)p.B * c * 2 <= sm_count())) c *= 2;
  switch (c) {
    case 1: return launch_sample_filters<T, 1>(p, st);
    case 2: return launch_sample_filters<T, 2>(p, st);
    case 4: return launch_sample_filters<T, 4>(p, st);
    default: return launch_sample_filters<T, 8>(p, st);
  }
}

}  // namespace arke

using namespace arke;

extern "C" int arke_b200_sample_tokens(const void* logits, int dtype, int64_t ld, int64_t B, int64_t V, const float* u,
                                       const float* temperature_row, float temperature, const int32_t* top_k_row,
                                       int64_t top_k, const float* top_p_row, float top_p, const float* min_p_row,
                                       float min_p, int64_t* token, float* logprob, void* stream) {
  if (B < 0 || B > (1 << 24) || V <= 0 || V > (1 << 20)) return set_error(ARKE_ERR_SHAPE, "sample_tokens: need rows >= 0 and 0 < V <= 2^20");
  if (ld < V) return set_error(ARKE_ERR_SHAPE, "sample_tokens: row stride smaller than V");
  if (dtype != ARKE_BF16 && dtype != ARKE_F16 && dtype != ARKE_F32) return set_error(ARKE_ERR_DTYPE, "sample_tokens: logits must be bf16, f16 or f32");
  if (!temperature_row && !(temperature >= 0.f)) return set_error(ARKE_ERR_ARG, "sample_tokens: the temperature must not be negative");
  if (!top_k_row && top_k < 0) return set_error(ARKE_ERR_ARG, "sample_tokens: top_k must not be negative (0 = all)");
  if (!top_p_row && !(top_p >= 0.f)) return set_error(ARKE_ERR_ARG, "sample_tokens: top_p must not be negative");
  if (!min_p_row && !(min_p >= 0.f && min_p <= 1.f)) return set_error(ARKE_ERR_ARG, "sample_tokens: min_p must lie in [0, 1]");
  if (B == 0) return ARKE_OK;
  if (!logits || !u || !token) return set_error(ARKE_ERR_ARG, "sample_tokens: null pointer");
  int rc = require_sm100("sample_tokens");
  if (rc != ARKE_OK) return rc;
  ARKE_API_ENTER("arke_b200_sample_tokens");
  SampleParams p{};
  p.x = static_cast<const char*>(logits);
  p.ld = ld;
  p.u = u;
  p.t_row = temperature_row;
  p.k_row = top_k_row;
  p.p_row = top_p_row;
  p.m_row = min_p_row;
  p.t = temperature;
  p.k = top_k < V ? (int)top_k : 0;
  p.p = top_p;
  p.m = min_p;
  p.token = token;
  p.logprob = logprob;
  p.B = (int)B;
  p.V = (int)V;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == ARKE_BF16) return launch_sample<__nv_bfloat16>(p, st);
  if (dtype == ARKE_F16) return launch_sample<__half>(p, st);
  return launch_sample<float>(p, st);
}
