// Grouped-query attention of a ragged batch over a paged key/value cache, for one or a few new
// tokens per sequence, with an optional prefix that all sequences share.
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = 2^(s_rj - m_r),   s_rj = q_r.k_j * scale * log2(e),   j < seen_r
//
// Rows.  The query rows that read the same keys are stacked: the n tokens x G = Hq / Hkv query heads
// of one sequence and key head, or, over the shared prefix, those of all sequences.  A "unit" is one
// block of R stacked rows of one key head and its keys; each key and value is read once per unit.
//
// Split.  The tiles (16 or 32 keys) of all units, prefix first, form one line; each warp takes an equal,
// contiguous share of it (beside tensor-core tiles: two sizes, see make_shares), computed on the device
// from kv_lens, so neither the host nor a captured graph has to know the lengths and a long sequence
// beside many short ones leaves no SM idle.  A unit that one warp covers is finished there; the others
// leave (m, l, o) partials in fp32 that a second small kernel joins in a fixed order.
//
// Tile.  Every warp streams its tiles through a private cp.async ring and nothing in the loop waits for
// another warp; the ring runs on into the next unit, so short sequences do not drain it.  S^T[keys,
// rows] = K Q^T by mma.sync m16n8k16 with the keys as M, so that 8 rows are a whole N tile and a single
// token of G <= 8 heads wastes little, and O^T += V^T P^T, whose B operand is the transposed S^T
// fragment (movmatrix).  P is split in two 16-bit parts (value and remainder), which keeps it exact to
// about 2^-17: the second product costs nothing while the kernel waits for HBM.  The running maximum
// moves only when it grows by more than 2^8, so almost no tile needs a shuffle or a rescale.  Sums,
// maxima and O are fp32.
//
// Bound: HBM.  Few rows make 2 * R flops per byte, far below the ridge, so tcgen05 with its 128-row
// tiles could only add latency here.  64 ragged sequences of up to 8192 positions (32 / 8 heads, D = 128,
// 1.25 GB): 200 us, 6.25 TB/s, 97 % of the measured copy rate; with the four warps of a CTA on one tile, a
// barrier per unit and a drained ring between units it was 222 us, and 256 short sequences (5 tiles of
// 64 keys) lost almost half their time.  Short calls are a chain of latencies (lengths, table, keys,
// partials, join: one sequence of 1000 positions 14 us in a graph, 4.1 MB).
#include "paged_att.cuh"
#include <limits.h>
#include <math.h>
#include <type_traits>

namespace arke {

constexpr int kPagThreads = 128;
constexpr int kPagWarps = kPagThreads / 32;

// Keys per tile: 8 KB of keys and values for both head sizes.  With 16 keys at D = 64 the instructions of a tile, not its
// 4 KB, set the pace (98 sequences of 2828 positions, 12 key heads: 171 us; with 32 keys within 9 us of the 132 us that
// the bytes take).
__host__ __device__ constexpr int pag_tile(int D) { return D == 128 ? 16 : 32; }

template <int D>
struct PagSmem {
  static constexpr int kStages = 3;                             // 24 KB in flight per warp, 192 KB per SM
  static constexpr int kTile = pag_tile(D);
  static constexpr int kRowBytes = D * 2;
  static constexpr int kHalfStage = kTile * kRowBytes;          // K or V of one tile
  static constexpr int kStage = 2 * kHalfStage;
  static constexpr int kWarp = kStages * kStage;
  static constexpr int kTotal = kPagWarps * kWarp;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two floats -> their 16-bit values (lo half = a) and the 16-bit values of what the rounding left
template <typename T>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    hi = pack_bf16x2(a, b);
    lo = pack_bf16x2(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
  } else {
    hi = pack_f16x2(a, b);
    float x, y;
    unpack_f16x2(hi, x, y);
    lo = pack_f16x2(a - x, b - y);
  }
}

// Where a warp stands on the line of tiles: a unit (sequence b, or -1 for the shared prefix; key head h; row
// block rb) and a tile of it.
struct Cursor {
  int b, h, rb, t;     // t: tile inside the unit
  int tiles, nrb;      // of every unit of this sequence
  int n, len;          // its tokens, the end of its keys
  __device__ __forceinline__ void open(const PagedAttParams& p, int seq, int R) {
    b = seq;
    const SeqWork w = seq_work(p, b);
    tiles = w.tiles;
    n = w.n;
    len = w.len;
    nrb = row_blocks(p, n, R);
  }
  // the first tile of the next unit; only called while there is one
  __device__ __forceinline__ void next_unit(const PagedAttParams& p, int R) {
    t = 0;
    if (++rb < nrb) return;
    rb = 0;
    if (++h < p.kv.Hkv) return;
    h = 0;
    do open(p, b + 1, R);
    while (tiles == 0 || nrb == 0);
  }
};

// This CTA's warp `w` in the order of the shares: early CTAs' before the others', and of few tiles one warp of every SM
// gets some before a second one does.
__device__ __forceinline__ long long worker_of(const PagedAttParams& p, int w) {
  const int block = blockIdx.x;
  if (block < p.early) return (long long)w * p.early + block;
  return (long long)kPagWarps * p.early + (long long)w * (p.grid - p.early) + (block - p.early);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kPagThreads, 2) paged_gqa_kernel(const PagedAttParams p) {
  using SM = PagSmem<D>;
  constexpr int R = 8 * NT;
  constexpr int KS = D / 16;               // k-steps of Q K^T and m-tiles of O^T
  constexpr int CH = D / 8;                // 16-byte chunks per row
  constexpr int KT = SM::kTile / 16;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ long long s_scan[kPagWarps];
  __shared__ long long s_base[kPagWarps];
  __shared__ long long s_first[kPagWarps];               // where this CTA's warps' shares begin
  __shared__ int s_seq[kPagWarps];
  __shared__ unsigned s_units[kPagWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();

  // ---- schedule: tiles in all, this warp's share, the unit it begins in
  const int pre_tiles = p.pre_tile ? 0 : (p.prefix + SM::kTile - 1) / SM::kTile;
  const int tokens = p.kv.B > 0 ? seq_begin_clamped(p.kv, p.kv.B) : 0;
  const int pre_rb = row_blocks(p, tokens, R);
  const long long pre_total = (long long)pre_tiles * pre_rb * p.kv.Hkv;
  long long total = pre_total;
  Shares shares{0, 0, 0};
  long long units = (long long)(pre_tiles > 0 ? pre_rb : 0) * p.kv.Hkv;
  long long w_first = 0;                                 // tiles of sequence `tid`
  unsigned u_first = 0;                                  // its units, of one head
  if (tid < p.kv.B) {
    const SeqWork sw = seq_work(p, tid);
    u_first = sw.tiles > 0 ? row_blocks(p, sw.n, R) : 0;
    w_first = (long long)sw.tiles * u_first * p.kv.Hkv;
  }
  for (int pass = 0; pass < 2; ++pass) {
    long long base = pre_total;
    for (int b0 = 0; b0 < p.kv.B; b0 += kPagThreads) {
      const int b = b0 + tid;
      long long w = w_first;
      unsigned u = u_first;
      if (b0 > 0) {
        w = u = 0;
        if (b < p.kv.B) {
          const SeqWork sw = seq_work(p, b);
          u = sw.tiles > 0 ? row_blocks(p, sw.n, R) : 0;
          w = (long long)sw.tiles * u * p.kv.Hkv;
        }
      }
      long long inc = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += v;
      }
      u = __reduce_add_sync(0xffffffffu, u);
      if (lane == 31) { s_scan[warp] = inc; s_units[warp] = u; }
      __syncthreads();
      long long end = base + inc;
      for (int i = 0; i < kPagWarps; ++i) {
        if (i < warp) end += s_scan[i];
        base += s_scan[i];
        if (!pass) units += (long long)s_units[i] * p.kv.Hkv;
      }
      const long long begin = end - w;
      if (pass) {
        if (w > 0)
          for (int i = 0; i < kPagWarps; ++i) {
            if (begin <= s_first[i] && s_first[i] < end) { s_seq[i] = b; s_base[i] = begin; }
          }
        if (blockIdx.x == 0 && b < p.kv.B && ARKE_CHK(b, b, p.kv.B)) p.sched[2 + b] = begin;
      }
      __syncthreads();
    }
    if (!pass) {
      total = base;
      shares = make_shares(p, total, units, kPagWarps, R);
      if (tid < kPagWarps) s_first[tid] = shares.first_of(worker_of(p, tid));
      __syncthreads();
    }
  }
  if (blockIdx.x == 0 && tid == 0) { p.sched[0] = shares.early; p.sched[1] = shares.other; }
  const long long worker = worker_of(p, warp);
  const long long pos0 = s_first[warp], mine = (int)blockIdx.x < p.early ? shares.early : shares.other;
  int left = (int)(pos0 >= total ? 0 : total - pos0 < mine ? total - pos0 : mine);      // tiles still to compute
  if (left > 0) {
    const uint32_t ring = smem_u32(smem) + warp * SM::kWarp;
    Cursor cur;
    long long within;
    if (pos0 < pre_total) {
      cur.b = -1;
      cur.tiles = pre_tiles;
      cur.nrb = pre_rb;
      cur.n = tokens;
      cur.len = prefix_data_end(p);
      within = pos0;
    } else {
      cur.open(p, s_seq[warp], R);
      within = pos0 - s_base[warp];
    }
    {
      const int unit = (int)(within / cur.tiles);
      cur.t = (int)(within - (long long)unit * cur.tiles);
      cur.h = unit / cur.nrb;
      cur.rb = unit - cur.h * cur.nrb;
    }

    // ---- loads run ahead of the products: lane l looks up the page of key l of a tile
    Cursor ahead = cur;
    int to_issue = left;
    bool bad = false;                                    // a missing page in the unit being computed
    unsigned bad_ring = 0;                               // one bit per stage
    int2 place;                                          // (page, row) of this lane's key, page -1: nothing to load
    // lane i: entry window_at + i of the sequence's table, so that a tile does not wait for a load of its own
    int window = 0, window_at = 0, window_end = -1;
    auto lookup = [&]() {
      const int key0 = (ahead.b >= 0 ? p.prefix : 0) + ahead.t * SM::kTile, key = key0 + (lane & (SM::kTile - 1));
      const int pg = key / p.kv.page_size;
      const int last = (min(key0 + SM::kTile, ahead.len) - 1) / p.kv.page_size;
      if (last >= window_end) {                          // the same in every lane
        window_at = key0 / p.kv.page_size;
        window_end = window_at + 32;
        const int at = window_at + lane;
        window = at < p.kv.max_pages && (ahead.b >= 0 || at < p.shared_pages) ? page_of(p, ahead.b, at) : 0;
      }
      const int id = __shfl_sync(0xffffffffu, window, (pg - window_at) & 31);
      place = make_int2(-1, 0);
      if (key < ahead.len) place = make_int2(id >= 0 && id < p.kv.num_pages ? id : -2, key - pg * p.kv.page_size);
    };
    lookup();
    auto issue = [&](int stage) {
      if (to_issue > 0) {
        const uint32_t dst = ring + stage * SM::kStage;
        const T* kbase = reinterpret_cast<const T*>(p.kv.k) + (int64_t)ahead.h * p.kv.ksh;
        const T* vbase = reinterpret_cast<const T*>(p.kv.v) + (int64_t)ahead.h * p.kv.vsh;
        const unsigned any = __any_sync(0xffffffffu, place.x == -2);
        bad_ring = (bad_ring & ~(1u << stage)) | (any << stage);
#pragma unroll
        for (int i = 0; i < SM::kTile * CH / 32; ++i) {
          const int c = i * 32 + lane;
          const int row = c / CH, ch = c % CH;
          const int page = __shfl_sync(0xffffffffu, place.x, row);
          const int prow = __shfl_sync(0xffffffffu, place.y, row);
          const bool ok = page >= 0;
          const int64_t ko = ok ? page * p.kv.ksp + prow * p.kv.ksr + ch * 8 : 0;
          const int64_t vo = ok ? page * p.kv.vsp + prow * p.kv.vsr + ch * 8 : 0;
          const uint32_t at = dst + row * SM::kRowBytes + ((ch ^ (row & 7)) << 4);
          const bool kok = ok && ARKE_CHK(ahead.h * p.kv.ksh + ko, ahead.h * p.kv.ksh + ko + 7, p.kv.k_ext);
          const bool vok = ok && ARKE_CHK(ahead.h * p.kv.vsh + vo, ahead.h * p.kv.vsh + vo + 7, p.kv.v_ext);
          cp_async16(at, kbase + ko, kok ? 16 : 0);          // 0 bytes: nothing is read, the row is zero
          cp_async16(at + SM::kHalfStage, vbase + vo, vok ? 16 : 0);
        }
        if (--to_issue > 0) {
          if (++ahead.t == ahead.tiles) {
            const int was = ahead.b;
            ahead.next_unit(p, R);
            if (ahead.b != was || ahead.t * SM::kTile / p.kv.page_size < window_at) window_end = -1;
          }
          lookup();
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < SM::kStages - 1; ++s) issue(s);
    int stage = 0, fill = SM::kStages - 1;

    while (left > 0) {
      // ---- a piece: tiles [cur.t, cur.t + m) of one unit
      const int m = min(left, cur.tiles - cur.t);
      const int tok0 = cur.b >= 0 ? seq_begin_clamped(p.kv, cur.b) : 0;
      const int row0 = cur.rb * R;
      const int rows = min(R, cur.n * p.G - row0);
      const int first = cur.b >= 0 ? p.prefix : 0;
      const bool whole = m == cur.tiles;
      // lane r: the call's row of stacked row r and what it may see
      int my_row = -1, my_seen = 0;                      // token * Hq + head
      {
        const int rr = row0 + min(lane, rows - 1), token = tok0 + rr / p.G;
        int seen;
        if (cur.b >= 0) {
          seen = p.causal ? cur.len - cur.n + (token - tok0) + 1 : cur.len;
        } else {
          seen = seen_by(p, find_sequence_lanes(p.kv, token), token);
        }
        if (lane < rows) {
          my_row = token * p.Hq + cur.h * p.G + rr % p.G;
          my_seen = seen;
        }
      }
      const int min_seen = __reduce_min_sync(0xffffffffu, lane < rows ? my_seen : INT_MAX);
      uint32_t qf[NT][KS][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int orow = __shfl_sync(0xffffffffu, my_row, (nt * 8 + (lane >> 2)) & 31);
        const int token = orow / p.Hq;
        const int64_t at = token * p.q_st + (int64_t)(orow - token * p.Hq) * p.q_sh;
        const bool ok = orow >= 0 && q_chk(p, at, D);
        const T* src = reinterpret_cast<const T*>(p.q) + at + 2 * (lane & 3);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          qf[nt][ks][0] = ok ? *reinterpret_cast<const uint32_t*>(src + ks * 16) : 0u;
          qf[nt][ks][1] = ok ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8) : 0u;
        }
      }
      float acc[KS][NT][4];
      float mx[NT][2], l[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mx[nt][0] = mx[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][nt][e] = 0.f;
      }
      bad = false;
      const int t_end = cur.t + m;
      for (; cur.t < t_end; ++cur.t) {
        cp_async_wait<SM::kStages - 2>();
        __syncwarp();
        bad |= (bad_ring >> stage) & 1;
        issue(fill);
        fill = fill + 1 == SM::kStages ? 0 : fill + 1;
        const uint32_t kst = ring + stage * SM::kStage;
        stage = stage + 1 == SM::kStages ? 0 : stage + 1;
        const int key = first + cur.t * SM::kTile;

        // S^T = K Q^T, 16 keys at a time
        float s[KT][NT][4];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) s[kt][nt][0] = s[kt][nt][1] = s[kt][nt][2] = s[kt][nt][3] = 0.f;
          const int row = kt * 16 + (lane & 15);
          const uint32_t rbase = kst + row * SM::kRowBytes;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t a[4];
            ldsm4(rbase + (((ks * 2 + (lane >> 4)) ^ (row & 7)) << 4), a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<T>(s[kt][nt], a, qf[nt][ks][0], qf[nt][ks][1]);
          }
        }
        // scores: element e belongs to key 16 kt + (lane / 4) + 8 * (e / 2) and row 2 * (lane % 4) + (e % 2)
        const bool mask = key + SM::kTile > min(cur.len, min_seen);
        bool grow = false;
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[kt][nt][e] *= p.scale_log2;
          if (mask) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int seen = min(cur.len, __shfl_sync(0xffffffffu, my_seen, (nt * 8 + 2 * (lane & 3) + e) & 31));
#pragma unroll
              for (int kt = 0; kt < KT; ++kt) {
                const int j = key + kt * 16 + (lane >> 2);
                if (j >= seen) s[kt][nt][e] = -INFINITY;
                if (j + 8 >= seen) s[kt][nt][e + 2] = -INFINITY;
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            top[nt][e] = fmaxf(s[0][nt][e], s[0][nt][e + 2]);
#pragma unroll
            for (int kt = 1; kt < KT; ++kt) top[nt][e] = fmaxf(top[nt][e], fmaxf(s[kt][nt][e], s[kt][nt][e + 2]));
            grow |= top[nt][e] > mx[nt][e] + 8.f;
          }
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float v = top[nt][e];
              v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
              v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
              v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
              v = fmaxf(v, mx[nt][e]);
              const float f = mx[nt][e] == -INFINITY ? 0.f : ex2_approx(mx[nt][e] - v);
              mx[nt][e] = v;
              l[nt][e] *= f;
#pragma unroll
              for (int i = 0; i < KS; ++i) {
                acc[i][nt][e] *= f;
                acc[i][nt][e + 2] *= f;
              }
            }
        }
        uint32_t hi[KT][NT][2], lo[KT][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float m0 = mx[nt][0] == -INFINITY ? 0.f : mx[nt][0], m1 = mx[nt][1] == -INFINITY ? 0.f : mx[nt][1];
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const float p0 = ex2_approx(s[kt][nt][0] - m0), p1 = ex2_approx(s[kt][nt][1] - m1);
            const float p2 = ex2_approx(s[kt][nt][2] - m0), p3 = ex2_approx(s[kt][nt][3] - m1);
            l[nt][0] += p0 + p2;
            l[nt][1] += p1 + p3;
            split_pair<T>(p0, p1, hi[kt][nt][0], lo[kt][nt][0]);
            split_pair<T>(p2, p3, hi[kt][nt][1], lo[kt][nt][1]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              hi[kt][nt][e] = movmatrix_t(hi[kt][nt][e]);
              lo[kt][nt][e] = movmatrix_t(lo[kt][nt][e]);
            }
          }
        }
        // O^T += V^T P^T
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const int row = kt * 16 + (lane & 7) + ((lane >> 4) << 3);
          const uint32_t rbase = kst + SM::kHalfStage + row * SM::kRowBytes;
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            uint32_t a[4];
            ldsm4_t(rbase + (((i * 2 + ((lane >> 3) & 1)) ^ (row & 7)) << 4), a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma16816<T>(acc[i][nt], a, hi[kt][nt][0], hi[kt][nt][1]);
              mma16816<T>(acc[i][nt], a, lo[kt][nt][0], lo[kt][nt][1]);
            }
          }
        }
      }
      left -= m;
      const bool broken = bad;                           // the same in every lane
      if (broken && lane == 0) atomicCAS(p.status, 0, KSTAT_BAD_INDEX);

      // ---- the piece's rows: finished, or (m, l, o) for the join
      const bool starts = t_end == m;                    // the piece begins where the unit does
      const bool final_here = whole && p.prefix == 0;
      const float nan = __int_as_float(0x7fc00000);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float inv[2];
        int orow[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 4);
          l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 8);
          l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], 16);
          if (broken) { l[nt][e] = nan; mx[nt][e] = 0.f; }
          inv[e] = broken ? nan : !final_here ? 1.f : l[nt][e] == 0.f ? 0.f : 1.f / l[nt][e];
          orow[e] = __shfl_sync(0xffffffffu, my_row, (nt * 8 + 2 * (lane & 3) + e) & 31);
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            acc[i][nt][e] *= inv[e];
            acc[i][nt][e + 2] *= inv[e];
          }
        }
        if (final_here) {
          // two heads' values of one d -> two d's of one head, so that four lanes store 16 bytes of a row
          const int to = __shfl_sync(0xffffffffu, my_row, (nt * 8 + (lane >> 2)) & 31);
          const bool ok = to >= 0 && ARKE_CHK((int64_t)to * D, (int64_t)to * D + D - 1, (int64_t)p.kv.T * p.Hq * D);
          T* dst = reinterpret_cast<T*>(p.o) + (int64_t)to * D + 2 * (lane & 3);
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              uint32_t w;
              if constexpr (std::is_same<T, __nv_bfloat16>::value) w = pack_bf16x2(acc[i][nt][2 * half], acc[i][nt][2 * half + 1]);
              else w = pack_f16x2(acc[i][nt][2 * half], acc[i][nt][2 * half + 1]);
              w = movmatrix_t(w);
              if (ok) *reinterpret_cast<uint32_t*>(dst + i * 16 + half * 8) = w;
            }
          if (p.lse && lane < 4)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (orow[e] >= 0 && ARKE_CHK(orow[e], orow[e], (int64_t)p.kv.T * p.Hq)) p.lse[orow[e]] = l[nt][e] == 0.f ? -INFINITY : (mx[nt][e] + log2f(l[nt][e])) * 0.6931471805599453f;
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            if (orow[e] < 0) continue;
            const int64_t slot = whole ? orow[e] + (cur.b >= 0 ? (int64_t)p.kv.T * p.Hq : 0)
                                       : (worker * 2 + (starts ? 1 : 0)) * R + nt * 8 + 2 * (lane & 3) + e;
            if (!ARKE_CHK(slot, slot, whole ? p.row_rows : p.part_rows)) continue;
            float* po = (whole ? p.row_o : p.part_o) + slot * D + (lane >> 2);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              po[i * 16] = acc[i][nt][e];
              po[i * 16 + 8] = acc[i][nt][e + 2];
            }
            if (lane < 4) *reinterpret_cast<float2*>((whole ? p.row_ml : p.part_ml) + slot * 2) = make_float2(mx[nt][e], l[nt][e]);
          }
        }
      }
      if (left > 0) cur.next_unit(p, R);
    }
    cp_async_wait<0>();
  }
  if (p.pre_tile || p.seq_tile) pdl_wait();           // this grid ends after the tensor-core tiles': the join waits for both
}

// Joins the partials of every row that the kernels above left open, and writes the rows that saw nothing.
// WARPS warps share a row (token, head), a contiguous part of its partials each; a warp reads 32 (m, l) at
// once, one per lane, then adds the rows up with several loads in flight.  Where rows are few their partials
// are many, and one warp would read them for longer than the keys took.
constexpr int kJoinThreads = 256;
template <typename T, int D, int WARPS>
__device__ __forceinline__ void join_row(const PagedAttParams& p, int R, int64_t row, float (*s_part)[D + 2], bool& waited) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31, share = WARPS > 1 ? threadIdx.x >> 5 : 0;
  const int64_t all = (int64_t)p.kv.T * p.Hq;
  const int token = (int)(row / p.Hq), head = (int)(row - (int64_t)token * p.Hq);
  const int h = head / p.G, g = head - h * p.G;
  const int b = find_sequence_warp(p.kv, token);
  float top = -INFINITY, sum = 0.f, v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = 0.f;
  const bool live = b >= 0 && b < p.kv.B;
  const int len = live ? len_at(p.kv, b) : 0;
  const bool bad = len < 0 || len > p.kv.max_pages * p.kv.page_size;
  SeqWork sw{0, 0, 0};
  int rr = 0;
  // the four kinds of pieces: tensor-core parts of the prefix and of the sequence, streamed ones of both
  int count[4] = {0, 0, 0, 0};
  int64_t lo[2] = {0, 0};
  int r[2] = {0, 0};
  bool whole[2] = {false, false};
  int dual[2] = {0, 0};                                 // tensor-core parts in two halves
  bool done = false;
  if (live && !bad) {
    sw = seq_work(p, b);
    rr = (token - seq_begin_clamped(p.kv, b)) * p.G + g;
    if (p.pre_tile) {
      const int rest = seq_begin_clamped(p.kv, p.kv.B) * p.G - (token * p.G + g) / kTileRows * kTileRows;
      dual[0] = unit_is_dual(p, false, rest);
      count[0] = p.pre_split << dual[0];
    }
    if (seq_in_tiles(p, sw.n)) {
      const int row0 = rr / kTileRows * kTileRows;
      const UnitKeys u = seq_unit_keys(p, sw, row0, kTileRows);
      if (u.end > u.first) {
        dual[1] = unit_is_dual(p, true, sw.n * p.G - row0);
        done = p.seq_split == 1 && p.prefix == 0 && !dual[1];
        count[1] = p.seq_split << dual[1];
      }
    }
  }
  if (!waited) pdl_wait();                              // everything below is written by the kernels before
  waited = true;
  if (done) return;                                     // by its tile
  if (live && !bad) {
    const Shares shares{p.sched[0], p.sched[1], (long long)p.early * kPagWarps};
    const int pre_tiles = p.pre_tile ? 0 : (p.prefix + p.tile - 1) / p.tile;
    if (pre_tiles > 0) {
      const int pr = token * p.G + g;
      const int nrb = row_blocks(p, seq_begin_clamped(p.kv, p.kv.B), R), rb = pr / R;
      const int64_t s0 = ((int64_t)h * nrb + rb) * pre_tiles;
      lo[0] = shares.warp_at(s0);
      count[2] = (int)(shares.warp_at(s0 + pre_tiles - 1) - lo[0]) + 1;
      r[0] = pr - rb * R;
      whole[0] = count[2] == 1;
    }
    if (sw.tiles > 0) {
      const int nrb = row_blocks(p, sw.n, R), rb = rr / R;
      const int64_t s0 = (ARKE_CHK(b, b, p.kv.B) ? p.sched[2 + b] : 0) + ((int64_t)h * nrb + rb) * sw.tiles;
      lo[1] = shares.warp_at(s0);
      count[3] = (int)(shares.warp_at(s0 + sw.tiles - 1) - lo[1]) + 1;
      r[1] = rr - rb * R;
      whole[1] = count[3] == 1;
      if (whole[1] && p.prefix == 0) return;          // written by the warp that covered it
    }
    const int all_pieces = count[0] + count[1] + count[2] + count[3];
    const int n = (int)((int64_t)all_pieces * (share + 1) / WARPS);       // this warp's end
    for (int i0 = (int)((int64_t)all_pieces * share / WARPS); i0 < n; i0 += 32) {
      int i = i0 + lane;
      const float* po = nullptr;
      float2 q = make_float2(-INFINITY, 0.f);
      if (i < n) {
        const float* pm;
        if (i < count[0] + count[1]) {
          const int kind = i >= count[0];
          const int s = i - (kind ? count[0] : 0), two = kind ? dual[1] : dual[0];
          int j0, j1;
          unit_steps(kind ? seq_unit_keys(p, sw, rr / kTileRows * kTileRows, kTileRows) : prefix_unit_keys(p), kind ? p.seq_split : p.pre_split,
                     s >> two, j0, j1);
          if (two && (s & 1)) ++j0;                     // the second half has the odd steps
          if (j0 < j1 && ARKE_CHK(s * all + row, s * all + row, p.tile_rows[kind])) po = (kind ? p.tile_o[1] : p.tile_o[0]) + (s * all + row) * D;
          pm = (kind ? p.tile_ml[1] : p.tile_ml[0]) + (s * all + row) * 2;
        } else {
          i -= count[0] + count[1];
          const int u = i >= count[2];
          const int64_t from = u ? lo[1] : lo[0], c = from + i - (u ? count[2] : 0);
          const bool one = u ? whole[1] : whole[0];
          const int64_t slot = one ? row + u * all : (c * 2 + (c == from ? 1 : 0)) * R + (u ? r[1] : r[0]);
          if (ARKE_CHK(slot, slot, one ? p.row_rows : p.part_rows)) po = (one ? p.row_o : p.part_o) + slot * D;
          pm = (one ? p.row_ml : p.part_ml) + slot * 2;
        }
        if (po) q = *reinterpret_cast<const float2*>(pm);
      }
      float m = q.x;
#pragma unroll
      for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      m = fmaxf(m, top);
      const float old = top == -INFINITY ? 0.f : ex2_approx(top - m);
      // no maximum but a sum: NaN scores
      const float f = q.x == -INFINITY ? (q.y == 0.f ? 0.f : 1.f) : ex2_approx(q.x - m);
      float part = f * q.y;
#pragma unroll
      for (int d = 16; d; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
      sum = sum * old + part;
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] *= old;
      top = m;
      const int here = min(32, n - i0);
#pragma unroll 8
      for (int k = 0; k < here; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        const float* pk = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(po), k));
        float x[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = 0.f;
        if (pk) {
          if constexpr (V == 4) *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(pk + lane * V);
          else *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(pk + lane * V);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = fmaf(fk, x[e], v[e]);
      }
    }
  } else if (bad) {
    sum = __int_as_float(0x7fc00000);                   // a length that the table cannot hold
    if (lane == 0) atomicCAS(p.status, 0, KSTAT_BAD_INDEX);
  }
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int e = 0; e < V; ++e) s_part[share][lane * V + e] = v[e];
    if (lane == 0) {
      s_part[share][D] = top;
      s_part[share][D + 1] = sum;
    }
    __syncthreads();
    if (share > 0) return;                              // one row to a CTA
    const float qm = lane < WARPS ? s_part[lane][D] : -INFINITY, ql = lane < WARPS ? s_part[lane][D + 1] : 0.f;
    top = qm;
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float f = qm == -INFINITY ? (ql == 0.f ? 0.f : 1.f) : ex2_approx(qm - top);
    sum = f * ql;
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float fw = __shfl_sync(0xffffffffu, f, w);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = fmaf(fw, s_part[w][lane * V + e], v[e]);
    }
  }
  if (!ARKE_CHK(row * D, row * D + D - 1, all * D)) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T out[V];
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = pag_round<T>(v[i] * inv);
  T* dst = reinterpret_cast<T*>(p.o) + row * D + lane * V;
  if constexpr (V == 4) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(out);
  else *reinterpret_cast<uint32_t*>(dst) = *reinterpret_cast<const uint32_t*>(out);
  if (p.lse && lane == 0) p.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(kJoinThreads) paged_gqa_join_kernel(const PagedAttParams p, int R) {
  __shared__ float s_part[WARPS > 1 ? WARPS : 1][D + 2];
  constexpr int rows = WARPS > 1 ? 1 : kJoinThreads / 32;              // at once
  bool waited = false;
  for (int64_t row = (int64_t)blockIdx.x * rows + (WARPS > 1 ? 0 : threadIdx.x >> 5); row < (int64_t)p.kv.T * p.Hq; row += (int64_t)gridDim.x * rows)
    join_row<T, D, WARPS>(p, R, row, s_part, waited);
}

// ---------------------------------------------------------------------------------------- host
constexpr int64_t kPrefixKB = 40 << 10;
static int pag_grid() {
  const int sms = sm_count();
  return 2 * (sms > 0 ? sms : 148);
}
// Whether the shared prefix gets units of its own.  They read it once for all sequences, but cost a launch of tiles and
// a second partial of every row; without them every sequence's units read it again, from L2.  Not worth it where a
// sequence has the rows to use what it reads, or where it is little.  Apart / together in us: 4 sequences behind 2048
// positions (24 MB saved) 19.0 / 17.9, 16 behind 512 (30 MB) 19.4 / 19.2, 6 behind 2048 (40 MB) 19.3 / 20.3, 16 behind
// 1024 (60 MB) 19.5 / 22.6, 128 behind 256 (127 MB) 23 / 35.
static bool split_prefix(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix) {
  const int64_t kb = tuning_options().paged_prefix_kb;
  return prefix > 0 && B > 1 && T * (Hq / Hkv) < B * (kTileRows / 2) && 
         (double)(B - 1) * (double)prefix * (double)(Hkv * D * 4) > (double)((kb > 0 ? kb : kPrefixKB) << 10);
}
struct PagLayout {
  size_t sched, part_o, part_ml, row_o, row_ml, tile_o[2], tile_ml[2], total;
  int64_t part_rows, row_rows, tile_rows[2];
};
static PagLayout pag_layout(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t prefix, int grid) {
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  if (!split_prefix(T, B, Hq, Hkv, D, prefix)) prefix = 0;
  PagLayout w;
  size_t at = 0;
  w.sched = at;   at += up(sizeof(int64_t) * (size_t)(2 + B));
  const size_t slots = 2 * (size_t)grid * kPagWarps * (T * (Hq / Hkv) <= 8 ? 8 : kFewRows);     // two per warp, of a block's rows
  w.part_o = at;  at += up(sizeof(float) * slots * (size_t)D);
  w.part_ml = at; at += up(sizeof(float) * slots * 2);
  const size_t rows = prefix > 0 ? (size_t)T * (size_t)Hq : 0;
  w.row_o = at;   at += up(sizeof(float) * 2 * rows * (size_t)D);
  w.row_ml = at;  at += up(sizeof(float) * 2 * rows * 2);
  int64_t tile[2];
  paged_tile_rows(T, B, Hq, Hkv, prefix, grid / 2, tile);
  for (int i = 0; i < 2; ++i) {
    w.tile_o[i] = at;  at += up(sizeof(float) * (size_t)tile[i] * (size_t)D);
    w.tile_ml[i] = at; at += up(sizeof(float) * (size_t)tile[i] * 2);
    w.tile_rows[i] = tile[i];
  }
  w.part_rows = (int64_t)slots;
  w.row_rows = 2 * (int64_t)rows;
  w.total = at;
  return w;
}

// stacked rows of an average sequence
static int64_t avg_rows(const PagedAttParams& p) { return ((int64_t)p.kv.T + p.kv.B - 1) / (p.kv.B > 0 ? p.kv.B : 1) * p.G; }

template <typename T, int D, int NT>
static int launch_paged(const PagedAttParams& p, cudaStream_t st) {
  using SM = PagSmem<D>;
  auto kern = paged_gqa_kernel<T, D, NT>;
  cudaError_t e = ensure_dynamic_smem(kern, SM::kTotal);
  if (e != cudaSuccess) return set_cuda_error("paged_gqa_fwd shared memory", e);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.grid);
  cfg.blockDim = dim3(kPagThreads);
  cfg.dynamicSmemBytes = SM::kTotal;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = p.pre_tile || p.seq_tile ? 1 : 0;    // beside the tensor-core tiles, on the SMs they leave
  e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return set_cuda_error("paged_gqa_fwd launch", e);
  const int64_t rows = (int64_t)p.kv.T * p.Hq;
  // A CTA for each row where the warps are many to a unit, and so the partials to a row, and the rows one wave.
  const int64_t units = (int64_t)p.kv.B * p.kv.Hkv * ((avg_rows(p) + 8 * NT - 1) / (8 * NT));
  const bool few = rows <= 1024 && (p.pre_tile || p.seq_tile || (int64_t)p.grid * kPagWarps >= 12 * units);
  cfg.gridDim = dim3((unsigned)(few ? rows : rows > 16 * (int64_t)p.grid ? 2 * p.grid : (rows + 7) / 8));   // at most four CTAs an SM
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  e = few ? cudaLaunchKernelEx(&cfg, paged_gqa_join_kernel<T, D, 8>, p, 8 * NT)
          : cudaLaunchKernelEx(&cfg, paged_gqa_join_kernel<T, D, 1>, p, 8 * NT);
  return e == cudaSuccess ? ARKE_OK : set_cuda_error("paged_gqa_fwd join launch", e);
}

template <typename T, int D>
static int dispatch_paged(const PagedAttParams& p, cudaStream_t st) {
  // Rows of a unit: the smallest block that holds an average sequence's rows (or, over a prefix,
  // as many as there are): fewer blocks re-read fewer keys, smaller ones compute fewer unused rows.
  int64_t rows = avg_rows(p);
  if (p.seq_tile && rows > kFewRows) rows = p.G;      // longer sequences are not this kernel's
  if (p.prefix > 0 && !p.pre_tile && (int64_t)p.kv.T * p.G > rows) rows = (int64_t)p.kv.T * p.G;
  if (rows <= 8) return launch_paged<T, D, 1>(p, st);
  if (rows <= 16) return launch_paged<T, D, 2>(p, st);
  return launch_paged<T, D, 4>(p, st);
}

}  // namespace arke

using namespace arke;

extern "C" size_t arke_b200_paged_gqa_workspace(int64_t T, int64_t batch, int64_t Hq, int64_t Hkv, int64_t D,
                                                int64_t shared_prefix) {
  if (T < 0 || batch < 0 || Hq <= 0 || Hkv <= 0 || D < 0 || shared_prefix < 0) return 0;
  return pag_layout(T, batch, Hq, Hkv, D, shared_prefix, pag_grid()).total;
}

extern "C" int arke_b200_paged_gqa_fwd(const void* q, int64_t q_stride_token, int64_t q_stride_head,
                                       const arke_b200_paged_kv* kv, void* o, float* lse, int64_t T, int64_t Hq,
                                       int64_t shared_prefix, int causal, float softmax_scale, void* workspace,
                                       size_t workspace_bytes, void* stream) {
  PagedAttParams p{};
  int rc = check_paged("paged_gqa_fwd", kv, T, Hq, &p.kv);
  if (rc != ARKE_OK) return rc;
  const int64_t D = kv->head_dim;
  if (D != 64 && D != 128) return set_error(ARKE_ERR_SHAPE, "paged_gqa_fwd: head_dim must be 64 or 128");
  if (shared_prefix < 0 || shared_prefix > kv->max_pages * kv->page_size)
    return set_error(ARKE_ERR_SHAPE, "paged_gqa_fwd: shared_prefix must lie within the block table");
  if (T * Hq * D > ((int64_t)1 << 40) || T * Hq > INT32_MAX) return set_error(ARKE_ERR_SHAPE, "paged_gqa_fwd: too many query rows");
  if (T == 0) return ARKE_OK;
  if (!q || !o) return set_error(ARKE_ERR_ARG, "paged_gqa_fwd: null pointer");
  auto al = [](const void* x, uintptr_t n) { return (reinterpret_cast<uintptr_t>(x) & (n - 1)) == 0; };
  if (!al(kv->k, 16) || !al(kv->v, 16) || !al(o, 16) || !al(q, 4) || (q_stride_token & 1) || (q_stride_head & 1) || p.kv.ksp % 8 ||
      p.kv.ksh % 8 || p.kv.ksr % 8 || p.kv.vsp % 8 || p.kv.vsh % 8 || p.kv.vsr % 8)
    return set_error(ARKE_ERR_ALIGN, "paged_gqa_fwd: caches and o must be 16-byte aligned with strides of whole 16 bytes, q 4-byte aligned");
  rc = require_sm100("paged_gqa_fwd");
  if (rc != ARKE_OK) return rc;
  ARKE_API_ENTER("arke_b200_paged_gqa_fwd");
  const int grid = pag_grid();
  const PagLayout w = pag_layout(T, kv->batch, Hq, kv->heads, D, shared_prefix, grid);
  if (!workspace || workspace_bytes < w.total) return set_error(ARKE_ERR_WORKSPACE, "paged_gqa_fwd: workspace too small");
  if (!al(workspace, 256)) return set_error(ARKE_ERR_ALIGN, "paged_gqa_fwd: the workspace must be 256-byte aligned");
  char* ws = static_cast<char*>(workspace);
  p.q = static_cast<const char*>(q);
  p.q_st = q_stride_token;
  p.q_sh = q_stride_head;
  p.o = static_cast<char*>(o);
  p.lse = lse;
  p.Hq = (int)Hq;
  p.G = (int)(Hq / kv->heads);
  // whole pages are shared; of a page that the prefix fills in part every sequence has its own
  p.shared_pages = kv->batch > 0 ? (int)(shared_prefix / kv->page_size) : 0;
  p.prefix = p.shared_pages * p.kv.page_size;
  if (!split_prefix(T, kv->batch, Hq, kv->heads, D, p.prefix)) p.prefix = 0;
  p.tile = pag_tile((int)D);
  p.causal = causal != 0;
  const float scale = softmax_scale > 0.f ? softmax_scale : 1.f / sqrtf((float)D);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.sched = reinterpret_cast<int64_t*>(ws + w.sched);
  p.part_o = reinterpret_cast<float*>(ws + w.part_o);
  p.part_ml = reinterpret_cast<float*>(ws + w.part_ml);
  p.row_o = reinterpret_cast<float*>(ws + w.row_o);
  p.row_ml = reinterpret_cast<float*>(ws + w.row_ml);
  p.grid = grid;
  const int64_t far_t = (T - 1) * q_stride_token, far_h = (Hq - 1) * q_stride_head;
  p.q_before = -((far_t < 0 ? far_t : 0) + (far_h < 0 ? far_h : 0));
  p.q_ext = p.q_before + (far_t > 0 ? far_t : 0) + (far_h > 0 ? far_h : 0) + D;
  p.part_rows = w.part_rows;
  p.row_rows = w.row_rows;
  for (int i = 0; i < 2; ++i) p.tile_rows[i] = w.tile_rows[i];
  p.status = kernel_status_ptr();
  if (!p.status) return ARKE_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  plan_paged_tiles(p, kv, grid / 2);
  if (p.pre_tile || p.seq_tile) {
    for (int i = 0; i < 2; ++i) {
      p.tile_o[i] = reinterpret_cast<float*>(ws + w.tile_o[i]);
      p.tile_ml[i] = reinterpret_cast<float*>(ws + w.tile_ml[i]);
    }
    rc = launch_paged_tiles(p, kv, st);
    if (rc == kNoTiles) p.pre_tile = p.seq_tile = p.early = p.early_tiles = 0;
    else if (rc != ARKE_OK) return rc;
  }
  if (kv->dtype == ARKE_BF16) return D == 128 ? dispatch_paged<__nv_bfloat16, 128>(p, st) : dispatch_paged<__nv_bfloat16, 64>(p, st);
  return D == 128 ? dispatch_paged<__half, 128>(p, st) : dispatch_paged<__half, 64>(p, st);
}
