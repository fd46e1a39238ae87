// What the kernels over a paged key/value cache share: the description of the batch and its pages,
// and the search for a token's sequence.
#pragma once
#include "common.cuh"
#include "capi_internal.h"

namespace arke {

// A ragged batch over a paged cache.  Sequence b owns the query tokens [cu_q[b], cu_q[b+1]) (or
// `uniform` tokens each when cu_q is null) and kv_lens[b] positions; position p lives in row
// p % page_size of page table[b][p / page_size].  Strides are in elements, the head dimension is
// contiguous.
struct PagedKV {
  const char* k;
  const char* v;
  int64_t ksp, ksh, ksr;   // page, head, row
  int64_t vsp, vsh, vsr;
  const int* table;
  int64_t ldt;
  const int* lens;
  const int* cu;
  int max_pages, num_pages, page_size;
  int B, uniform, T;       // T: query rows of the call, those behind the last sequence included
  int max_new;             // most query rows of a sequence as the caller knows it, 0 = unknown
  int Hkv;
  int64_t k_ext, v_ext;    // elements the caches span (checked build)
};

// Entries of the batch's description (the bounds are the checked build's).
__device__ __forceinline__ int cu_at(const PagedKV& p, int b) { return ARKE_CHK(b, b, p.B + 1) ? p.cu[b] : 0; }
__device__ __forceinline__ int len_at(const PagedKV& p, int b) { return ARKE_CHK(b, b, p.B) ? p.lens[b] : 0; }
__device__ __forceinline__ int table_at(const PagedKV& p, int b, int page) {
  return ARKE_CHK(b, b, p.B) && ARKE_CHK(page, page, p.max_pages) ? p.table[b * p.ldt + page] : -1;
}

__device__ __forceinline__ int seq_begin(const PagedKV& p, int b) { return p.cu ? cu_at(p, b) : b * p.uniform; }

// cu_q as the kernels use it: clamped to [0, T], so that no offset of a corrupt table leaves the call's rows
__device__ __forceinline__ int seq_begin_clamped(const PagedKV& p, int b) {
  const int s = seq_begin(p, b);
  return s < 0 ? 0 : s > p.T ? p.T : s;
}

// Sequence that owns query row t, for a whole warp with the same t: the last b with cu_q[b] <= t,
// found 32 entries at a time; B when t lies behind the last sequence, -1 in front of the first.
__device__ __forceinline__ int find_sequence_warp(const PagedKV& p, int t) {
  if (p.cu == nullptr) return p.uniform > 0 ? min(t / p.uniform, p.B) : p.B;
  const int lane = threadIdx.x & 31;
  // number of entries of cu_q[0..B] that are <= t; cu_q never decreases, so a 32-ary search finds it
  int lo = 0, hi = p.B + 1;                      // answer in [lo, hi]
  while (hi - lo > 0) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + (lane + 1) * step - 1;   // last entry of this lane's part
    const bool le = at < hi && cu_at(p, at) <= t;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int full = m == 0xffffffffu ? 32 : __ffs(~m) - 1;   // parts that lie at or below t altogether
    lo = lo + full * step;
    if (lo > hi) lo = hi;
    if (step == 1) break;
    hi = min(hi, lo + step - 1);
  }
  return lo - 1;
}

// The same for every lane of a warp with its own t, which never decreases from lane to lane: one search for the
// first lane's, then each walks on.
__device__ __forceinline__ int find_sequence_lanes(const PagedKV& p, int t) {
  if (p.cu == nullptr) return p.uniform > 0 ? min(t / p.uniform, p.B) : p.B;
  int b = find_sequence_warp(p, __shfl_sync(0xffffffffu, t, 0));
  while (b < p.B && cu_at(p, b + 1) <= t) ++b;
  return b;
}

int check_paged(const char* op, const arke_b200_paged_kv* d, int64_t T, int64_t Hq, PagedKV* out);

}  // namespace arke
