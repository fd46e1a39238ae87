// Appending to a paged key/value cache: the packed projections of a ragged batch are cut into
// heads, queries and keys are rotated to their positions, and keys and values go to the pages of
// their sequence — one HBM-bound pass that reads and writes each element once.
//
//   token i of sequence b (n new tokens, L positions after the append) has position p = L - n + i
//   y[:D/2] = x1 cos_p - x2 sin_p,   y[D/2:] = x2 cos_p + x1 sin_p      (fp32, one rounding)
//   key and value go to row p % page_size of page table[b][p / page_size]
//
// Unlike `rope`, which rounds every product to the 16-bit type as the interpreter does, products
// and sums stay in fp32 here and the result is rounded once: the cache is read for the rest of the
// sequence's life, and half a step is the least that 16 bits can lose.
#include "paged.cuh"
#include <stdio.h>

namespace arke {

struct AppendParams {
  PagedKV kv;
  const char* x;
  int64_t ldx;
  const char* cos;
  const char* sin;
  int64_t table_rows;
  const int* positions;   // rotation position of each query row, or null: its position in the sequence
  char* q;
  int Hq, D, T;
  int blocks_per_token;
  int* status;
};

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// Where one head of one token goes.  `rotate` is false for values; nullptr: nowhere.
struct AppendPlace {
  int seq;             // kv.B or -1: a row of no sequence
  int64_t rot;         // row of the cos / sin tables, -1 = outside them
  int64_t page;        // physical page, -1 = none
  int row;             // row inside the page
};

__device__ __forceinline__ AppendPlace append_place(const AppendParams& p, int t, int b) {
  AppendPlace a;
  a.seq = b;
  a.rot = -1;
  a.page = -1;
  a.row = 0;
  if (b < 0 || b >= p.kv.B) { a.seq = -1; return a; }
  const int s0 = seq_begin(p.kv, b), s1 = seq_begin(p.kv, b + 1);
  const int64_t pos = (int64_t)len_at(p.kv, b) - (s1 - s0) + (t - s0);
  const int64_t rot = p.positions ? (ARKE_CHK(t, t, p.T) ? (int64_t)p.positions[t] : -1) : pos;
  if (rot >= 0 && rot < p.table_rows) a.rot = rot;
  if (pos >= 0 && pos < (int64_t)p.kv.max_pages * p.kv.page_size) {
    const int pg = (int)(pos / p.kv.page_size);
    const int id = table_at(p.kv, b, pg);
    if (id >= 0 && id < p.kv.num_pages) { a.page = id; a.row = (int)(pos - (int64_t)pg * p.kv.page_size); }
  }
  return a;
}

template <typename T>
__device__ __forceinline__ T* append_dst(const AppendParams& p, const AppendPlace& a, int t, int h) {
  if (h < p.Hq) return reinterpret_cast<T*>(p.q) + ((int64_t)t * p.Hq + h) * p.D;
  if (a.page < 0 || a.rot < 0) return nullptr;
  const int hk = h - p.Hq;
  if (hk < p.kv.Hkv)
    return reinterpret_cast<T*>(const_cast<char*>(p.kv.k)) + a.page * p.kv.ksp + hk * p.kv.ksh + a.row * p.kv.ksr;
  return reinterpret_cast<T*>(const_cast<char*>(p.kv.v)) + a.page * p.kv.vsp + (hk - p.kv.Hkv) * p.kv.vsh + a.row * p.kv.vsr;
}

#ifdef ARKE_B200_CHECKED
template <typename T>
__device__ __forceinline__ bool append_chk(const AppendParams& p, const T* dst, int t, int h, int j, int n) {
  const int htot = p.Hq + 2 * p.kv.Hkv;
  const int half = p.D >> 1;
  const long long so = (long long)t * p.ldx + (long long)h * p.D + j;
  bool ok = ARKE_CHK(so, so + half + n - 1, span_elems(p.T, (long long)htot * p.D, p.ldx));
  if (h < p.Hq) {
    const long long o = dst - reinterpret_cast<const T*>(p.q);
    return ok && ARKE_CHK(o + j, o + j + half + n - 1, (long long)p.T * p.Hq * p.D);
  }
  const bool isk = h < p.Hq + p.kv.Hkv;
  const long long o = dst - reinterpret_cast<const T*>(isk ? p.kv.k : p.kv.v);
  return ok && ARKE_CHK(o + j, o + j + half + n - 1, isk ? p.kv.k_ext : p.kv.v_ext);
}
#define ARKE_APPEND_CHK(p, dst, t, h, j, n) append_chk<T>(p, dst, t, h, j, n)
#else
#define ARKE_APPEND_CHK(p, dst, t, h, j, n) (true)
#endif
// n elements from x's (t, h, j) on, and half a head further; n angles of row `rot`
__device__ __forceinline__ bool append_chk_x(const AppendParams& p, int t, int h, int j, int n) {
  [[maybe_unused]] const long long so = (long long)t * p.ldx + (long long)h * p.D + j;
  return ARKE_CHK(so, so + (p.D >> 1) + n - 1, span_elems(p.T, (long long)(p.Hq + 2 * p.kv.Hkv) * p.D, p.ldx));
}
__device__ __forceinline__ bool append_chk_angle(const AppendParams& p, int64_t rot, int j, int n) {
  [[maybe_unused]] const long long at = rot * (p.D >> 1) + j;
  return ARKE_CHK(at, at + n - 1, p.table_rows * (p.D >> 1));
}

template <typename TT>
__device__ __forceinline__ void load_table(const TT* src, float (&v)[8]) {
  if constexpr (sizeof(TT) == 4) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(src)), b = __ldg(reinterpret_cast<const float4*>(src) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(src));
    const TT* e = reinterpret_cast<const TT*>(&a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
  }
}

// One unit = 8 elements of the first half of a head and the same 8 of the second half; a thread takes UPT units, and
// a block never spans two tokens.  The loads of the row are under way while the warp looks for the token's sequence,
// page and angles, four loads that wait for one another: what bounds long prompts is how many bytes a block has in
// flight meanwhile (6000 tokens of 6144 f16 values, 3 units a thread instead of 1: 68.5 -> 57.9 us, 6.2 TB/s).
template <typename T, typename TT, int UPT>
__global__ void __launch_bounds__(128) paged_append_vec_kernel(const AppendParams p) {
  const int t = blockIdx.x / p.blocks_per_token;
  const int part = blockIdx.x - t * p.blocks_per_token;
  const int half = p.D >> 1, vpu = half / 8, htot = p.Hq + 2 * p.kv.Hkv;
  const T* row = reinterpret_cast<const T*>(p.x) + (int64_t)t * p.ldx;
  int h[UPT], j[UPT];
  uint4 a[UPT], b[UPT];
#pragma unroll
  for (int u = 0; u < UPT; ++u) {
    const int idx = (part * UPT + u) * 128 + threadIdx.x;
    h[u] = idx / vpu;
    j[u] = (idx - h[u] * vpu) * 8;
    a[u] = b[u] = make_uint4(0, 0, 0, 0);
    if (h[u] < htot && append_chk_x(p, t, h[u], j[u], 8)) {
      const T* src = row + h[u] * p.D + j[u];
      a[u] = __ldcs(reinterpret_cast<const uint4*>(src));
      b[u] = __ldcs(reinterpret_cast<const uint4*>(src + half));
    }
  }
  const AppendPlace at = append_place(p, t, find_sequence_warp(p.kv, t));
  if (at.seq >= 0 && (at.page < 0 || at.rot < 0) && threadIdx.x == 0 && part == 0) atomicCAS(p.status, 0, KSTAT_BAD_INDEX);
  float c[8], s[8];
  int have = -1;                                 // angles in registers: one load for all units where 128 is a multiple of vpu
#pragma unroll
  for (int u = 0; u < UPT; ++u) {
    if (h[u] >= htot) continue;
    T* dst = append_dst<T>(p, at, t, h[u]);
    if (at.seq < 0) {                            // a row behind the last sequence: q is zero, nothing is stored
      if (h[u] < p.Hq && ARKE_APPEND_CHK(p, dst, t, h[u], j[u], 8)) {
        *reinterpret_cast<uint4*>(dst + j[u]) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + j[u] + half) = make_uint4(0, 0, 0, 0);
      }
      continue;
    }
    if (dst == nullptr || !ARKE_APPEND_CHK(p, dst, t, h[u], j[u], 8)) continue;
    if (h[u] < p.Hq + p.kv.Hkv) {
      if (have != j[u]) {
        have = j[u];
        if (at.rot >= 0 && append_chk_angle(p, at.rot, j[u], 8)) {
          load_table<TT>(reinterpret_cast<const TT*>(p.cos) + at.rot * half + j[u], c);
          load_table<TT>(reinterpret_cast<const TT*>(p.sin) + at.rot * half + j[u], s);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
        }
      }
      const T* x1 = reinterpret_cast<const T*>(&a[u]);
      const T* x2 = reinterpret_cast<const T*>(&b[u]);
      uint4 o1, o2;
      T* y1 = reinterpret_cast<T*>(&o1);
      T* y2 = reinterpret_cast<T*>(&o2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = to_f32(x1[i]), w = to_f32(x2[i]);
        y1[i] = from_f32<T>(fmaf(x, c[i], -(w * s[i])));
        y2[i] = from_f32<T>(fmaf(w, c[i], x * s[i]));
      }
      a[u] = o1;
      b[u] = o2;
    }
    *reinterpret_cast<uint4*>(dst + j[u]) = a[u];        // plain stores: attention reads these next (L2)
    *reinterpret_cast<uint4*>(dst + j[u] + half) = b[u];
  }
}

// Any even head dimension, any alignment: one element pair per thread, two bytes at a time.  6000 tokens of 32 / 8 heads
// of 120, or of 128 at an odd offset: 161 and 169 us, 0.87 TB/s, against 28.7 us of the kernel above; 256 tokens 9.6
// against 4.1 us.  Bound by the loads' number.  No path of this library makes such rows (its projections are contiguous
// with heads of 64 and 128); who has long ones copies them to an aligned buffer first.
template <typename T, typename TT>
__global__ void __launch_bounds__(128) paged_append_scalar_kernel(const AppendParams p) {
  const int t = blockIdx.x / p.blocks_per_token;
  const int part = blockIdx.x - t * p.blocks_per_token;
  const int half = p.D >> 1, htot = p.Hq + 2 * p.kv.Hkv;
  const int idx = part * 128 + threadIdx.x;
  const int h = idx / half, j = idx - h * half;
  const AppendPlace at = append_place(p, t, find_sequence_warp(p.kv, t));
  if (h >= htot) return;
  T* dst = append_dst<T>(p, at, t, h);
  if (at.seq < 0) {
    if (h < p.Hq && ARKE_APPEND_CHK(p, dst, t, h, j, 1)) dst[j] = dst[j + half] = from_f32<T>(0.f);
    return;
  }
  if ((at.page < 0 || at.rot < 0) && threadIdx.x == 0 && part == 0) atomicCAS(p.status, 0, KSTAT_BAD_INDEX);
  if (dst == nullptr || !ARKE_APPEND_CHK(p, dst, t, h, j, 1)) return;
  const T* src = reinterpret_cast<const T*>(p.x) + (int64_t)t * p.ldx + (int64_t)h * p.D + j;
  T a = src[0], b = src[half];
  if (h < p.Hq + p.kv.Hkv) {
    float c = __int_as_float(0x7fc00000), s = c;
    if (at.rot >= 0 && append_chk_angle(p, at.rot, j, 1)) {
      c = to_f32(reinterpret_cast<const TT*>(p.cos)[at.rot * half + j]);
      s = to_f32(reinterpret_cast<const TT*>(p.sin)[at.rot * half + j]);
    }
    const float u = to_f32(a), w = to_f32(b);
    a = from_f32<T>(fmaf(u, c, -(w * s)));
    b = from_f32<T>(fmaf(w, c, u * s));
  }
  dst[j] = a;
  dst[j + half] = b;
}

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, typename TT>
static int launch_append(AppendParams& p, cudaStream_t st) {
  const int half = p.D / 2, htot = p.Hq + 2 * p.kv.Hkv;
  const bool vec = half % 8 == 0 && p.ldx % 8 == 0 && p.kv.ksp % 8 == 0 && p.kv.ksh % 8 == 0 && p.kv.ksr % 8 == 0 &&
                   p.kv.vsp % 8 == 0 && p.kv.vsh % 8 == 0 && p.kv.vsr % 8 == 0 && aligned16(p.x) && aligned16(p.cos) &&
                   aligned16(p.sin) && aligned16(p.q) && aligned16(p.kv.k) && aligned16(p.kv.v);
  const int64_t units = (int64_t)htot * (vec ? half / 8 : half);
  // Units per thread: one while that leaves SMs without a block; else what pads the token least, the most of equals.
  int upt = 1;
  if (vec && p.T * units >= (int64_t)sm_count() * 2048) {
    int64_t least = INT64_MAX;
    for (int n = 4; n >= 1; --n) {
      const int64_t padded = (units + 128 * n - 1) / (128 * n) * 128 * n;
      if (padded < least) { least = padded; upt = n; }
    }
  }
  p.blocks_per_token = (int)((units + 128 * upt - 1) / (128 * upt));
  const int64_t blocks = (int64_t)p.T * p.blocks_per_token;
  if (blocks > 0x7fffffffLL) return set_error(ARKE_ERR_SHAPE, "qkv_rope_paged_append: too many elements for one launch");
  if (!vec) paged_append_scalar_kernel<T, TT><<<(unsigned)blocks, 128, 0, st>>>(p);
  else if (upt == 1) paged_append_vec_kernel<T, TT, 1><<<(unsigned)blocks, 128, 0, st>>>(p);
  else if (upt == 2) paged_append_vec_kernel<T, TT, 2><<<(unsigned)blocks, 128, 0, st>>>(p);
  else if (upt == 3) paged_append_vec_kernel<T, TT, 3><<<(unsigned)blocks, 128, 0, st>>>(p);
  else paged_append_vec_kernel<T, TT, 4><<<(unsigned)blocks, 128, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ARKE_OK : set_cuda_error("qkv_rope_paged_append launch", e);
}

// Host-side checks of a cache description that both paged entry points make.
int check_paged(const char* op, const arke_b200_paged_kv* d, int64_t T, int64_t Hq, PagedKV* out) {
  char buf[256];
  auto fail = [&](int code, const char* what) {
    snprintf(buf, sizeof(buf), "%s: %s", op, what);
    return set_error(code, buf);
  };
  if (!d) return fail(ARKE_ERR_ARG, "null cache description");
  if (d->dtype != ARKE_BF16 && d->dtype != ARKE_F16) return fail(ARKE_ERR_DTYPE, "the cache must be bf16 or f16");
  if (T < 0 || T > (1 << 24) || d->batch < 0 || d->batch > (1 << 24)) return fail(ARKE_ERR_SHAPE, "token or sequence count out of range");
  if (d->heads <= 0 || Hq <= 0 || Hq > 65535 || d->heads > 65535 || Hq % d->heads != 0)
    return fail(ARKE_ERR_SHAPE, "the query heads must be a positive multiple of the key heads");
  if (d->head_dim <= 0 || (d->head_dim & 1) || d->head_dim > 1024) return fail(ARKE_ERR_SHAPE, "head_dim must be even and at most 1024");
  if (d->page_size <= 0 || d->page_size > (1 << 20) || d->num_pages < 0 || d->num_pages > INT32_MAX || d->max_pages < 0 ||
      d->max_pages > (1 << 30) / d->page_size)
    return fail(ARKE_ERR_SHAPE, "page size, page count or table width out of range");
  if (d->ld_table < d->max_pages) return fail(ARKE_ERR_SHAPE, "table row stride smaller than its width");
  const int64_t lim = (int64_t)1 << 46;
  for (int64_t s : {d->k_stride_page, d->k_stride_head, d->k_stride_row, d->v_stride_page, d->v_stride_head, d->v_stride_row})
    if (s < 0 || s > lim) return fail(ARKE_ERR_SHAPE, "cache strides must not be negative");
  if (!d->cu_q && d->batch > 0 && T % d->batch != 0) return fail(ARKE_ERR_SHAPE, "without cu_q every sequence has T / batch tokens, which must be a whole number");
  if (d->batch > 0 && !d->kv_lens) return fail(ARKE_ERR_ARG, "null kv_lens");
  if (d->batch > 0 && d->max_pages > 0 && !d->block_table) return fail(ARKE_ERR_ARG, "null block table");
  if (d->num_pages > 0 && (!d->k || !d->v)) return fail(ARKE_ERR_ARG, "null cache");
  PagedKV p{};
  p.k = static_cast<const char*>(d->k);
  p.v = static_cast<const char*>(d->v);
  p.ksp = d->k_stride_page; p.ksh = d->k_stride_head; p.ksr = d->k_stride_row;
  p.vsp = d->v_stride_page; p.vsh = d->v_stride_head; p.vsr = d->v_stride_row;
  p.table = d->block_table;
  p.ldt = d->ld_table;
  p.lens = d->kv_lens;
  p.cu = d->cu_q;
  p.max_pages = (int)d->max_pages;
  p.num_pages = (int)d->num_pages;
  p.page_size = (int)d->page_size;
  p.B = (int)d->batch;
  p.T = (int)T;
  p.max_new = d->max_new > 0 ? d->max_new : 0;
  p.uniform = d->batch > 0 ? (int)(T / d->batch) : 0;
  p.Hkv = (int)d->heads;
  if (d->num_pages > 0) {
    p.k_ext = (d->num_pages - 1) * p.ksp + (d->heads - 1) * p.ksh + (d->page_size - 1) * p.ksr + d->head_dim;
    p.v_ext = (d->num_pages - 1) * p.vsp + (d->heads - 1) * p.vsh + (d->page_size - 1) * p.vsr + d->head_dim;
  }
  *out = p;
  return ARKE_OK;
}

}  // namespace arke

using namespace arke;

extern "C" int arke_b200_qkv_rope_paged_append(const void* qkv, int64_t ld, const void* cos, const void* sin, int table_dtype,
                                               int64_t table_rows, const int32_t* positions, const arke_b200_paged_kv* kv,
                                               void* q, int64_t T, int64_t Hq, void* stream) {
  AppendParams p{};
  int rc = check_paged("qkv_rope_paged_append", kv, T, Hq, &p.kv);
  if (rc != ARKE_OK) return rc;
  const int64_t D = kv->head_dim, W = (Hq + 2 * kv->heads) * D;
  if ((kv->num_pages > 1 && (p.kv.ksp == 0 || p.kv.vsp == 0)) || (kv->heads > 1 && (p.kv.ksh == 0 || p.kv.vsh == 0)) ||
      (kv->page_size > 1 && (p.kv.ksr == 0 || p.kv.vsr == 0)))
    return set_error(ARKE_ERR_SHAPE, "qkv_rope_paged_append: rows of an expanded cache share their memory");
  if (ld < W) return set_error(ARKE_ERR_SHAPE, "qkv_rope_paged_append: row stride smaller than (Hq + 2 Hkv) * D");
  if (table_rows < 0) return set_error(ARKE_ERR_SHAPE, "qkv_rope_paged_append: negative table length");
  if (table_dtype != ARKE_F32 && table_dtype != kv->dtype)
    return set_error(ARKE_ERR_DTYPE, "qkv_rope_paged_append: cos and sin must be f32 or have the type of the cache");
  if (T == 0) return ARKE_OK;
  if (!qkv || !cos || !sin || !q) return set_error(ARKE_ERR_ARG, "qkv_rope_paged_append: null pointer");
  rc = require_sm100("qkv_rope_paged_append");
  if (rc != ARKE_OK) return rc;
  ARKE_API_ENTER("arke_b200_qkv_rope_paged_append");
  p.x = static_cast<const char*>(qkv);
  p.ldx = ld;
  p.cos = static_cast<const char*>(cos);
  p.sin = static_cast<const char*>(sin);
  p.table_rows = table_rows;
  p.positions = positions;
  p.q = static_cast<char*>(q);
  p.Hq = (int)Hq;
  p.D = (int)D;
  p.T = (int)T;
  p.status = kernel_status_ptr();
  if (!p.status) return ARKE_ERR_CUDA;
  cudaStream_t st = (cudaStream_t)stream;
  if (kv->dtype == ARKE_BF16)
    return table_dtype == ARKE_F32 ? launch_append<__nv_bfloat16, float>(p, st) : launch_append<__nv_bfloat16, __nv_bfloat16>(p, st);
  return table_dtype == ARKE_F32 ? launch_append<__half, float>(p, st) : launch_append<__half, __half>(p, st);
}
