// What the two attention kernels over a paged cache share: parameters and the division of the work.
#pragma once
#include "paged.cuh"

namespace arke {

constexpr int kFewRows = 32;        // most stacked rows that the streaming kernel takes in one unit
constexpr int kFewPrefixRows = 8;   // over a prefix all rows share the keys, and the partials of many would be many
constexpr int kTileRows = 256;      // rows of a tensor-core unit: two 128-row tiles
constexpr int kTileKeys = 128;

struct PagedAttParams {
  PagedKV kv;
  const char* q;
  int64_t q_st, q_sh;
  char* o;
  float* lse;
  int Hq, G;
  int prefix;          // positions that units of their own read once for all
  int shared_pages;    // pages that every sequence reads through row 0 of the table
  int tile;            // keys per tile of the streaming kernel
  int causal;
  float scale_log2;
  // workspace
  int64_t* sched;      // [0], [1] tiles per warp of an early and of another CTA, [2 + b] first tile of sequence b
  float* part_o;       // [2 * warps][R][D]
  float* part_ml;      // [2 * warps][R][2]
  float* row_o;        // [2][T * Hq][D]   units that one warp covers but another unit is joined with: prefix, own keys
  float* row_ml;       // [2][T * Hq][2]
  int grid;
  // the 128-row tensor-core tiles (paged_tile.cu)
  int pre_tile, seq_tile;     // whether they take the prefix, and the sequences with more than kFewRows rows
  int pre_split, seq_split;   // CTAs that share the keys of a unit
  int early, early_tiles;     // CTAs of the streaming kernel that run beside the tiles, and what a warp of theirs does meanwhile
  int seq_dual;               // whether sequences' units of one query tile use both pipelines (the prefix's always do)
  float* tile_o[2];           // [2 * split][T * Hq][D]: prefix, sequences
  float* tile_ml[2];          // [2 * split][T * Hq][2]
  int* status;
  // what the checked build holds every access against: q's first element before its pointer and elements from there on,
  // rows of the workspace's parts
  int64_t q_before, q_ext;
  int64_t part_rows, row_rows, tile_rows[2];
};
// n elements of q from offset `at` on
__device__ __forceinline__ bool q_chk(const PagedAttParams& p, int64_t at, int n) { return ARKE_CHK(at + p.q_before, at + p.q_before + n - 1, p.q_ext); }

// Keys of sequence b behind the shared prefix (0 when there is none), in tiles.
struct SeqWork {
  int n, len, tiles;       // new tokens, positions (clamped to what the table can hold), tiles
};
__device__ __forceinline__ bool seq_in_tiles(const PagedAttParams& p, int n) { return p.seq_tile && (int64_t)n * p.G > kFewRows; }
__device__ __forceinline__ SeqWork seq_work(const PagedAttParams& p, int b) {
  SeqWork w;
  const int s0 = seq_begin_clamped(p.kv, b), s1 = seq_begin_clamped(p.kv, b + 1);
  w.n = s1 > s0 ? s1 - s0 : 0;
  const int cap = p.kv.max_pages * p.kv.page_size;
  const int len = len_at(p.kv, b);
  w.len = len < 0 ? 0 : len > cap ? cap : len;
  w.tiles = w.len > p.prefix && !seq_in_tiles(p, w.n) ? (w.len - p.prefix + p.tile - 1) / p.tile : 0;
  return w;
}
// Where the data of a shared prefix ends, for a whole warp: with its longest sequence at the latest (of those with a token
// and a length within its range).  What lies behind that nobody has, and it may hold anything; it is read as if it were
// not there, while units and their steps go by the whole prefix, so that nothing waits for the lengths.
__device__ __forceinline__ int prefix_data_end(const PagedAttParams& p) {
  const int cap = p.kv.max_pages * p.kv.page_size;
  int longest = 0;
  for (int b = threadIdx.x & 31; b < p.kv.B; b += 32) {
    const int len = len_at(p.kv, b);
    if (len <= cap && seq_begin_clamped(p.kv, b + 1) > seq_begin_clamped(p.kv, b)) longest = max(longest, len);
  }
  return min(__reduce_max_sync(0xffffffffu, longest), p.prefix);
}
// Entry `page` of sequence b's row of the block table (b = -1: the shared prefix).
__device__ __forceinline__ int page_of(const PagedAttParams& p, int b, int page) {
  return table_at(p.kv, page < p.shared_pages ? 0 : b, page);
}
// Positions that query row `token` of sequence b sees (0: no such sequence).
__device__ __forceinline__ int seen_by(const PagedAttParams& p, int b, int token) {
  if (b < 0 || b >= p.kv.B) return 0;
  const SeqWork w = seq_work(p, b);
  return p.causal ? w.len - w.n + (token - seq_begin_clamped(p.kv, b)) + 1 : w.len;
}
__device__ __forceinline__ int row_blocks(const PagedAttParams& p, int n, int R) { return (int)(((int64_t)n * p.G + R - 1) / R); }

template <typename T> __device__ __forceinline__ T pag_round(float v);
template <> __device__ __forceinline__ __nv_bfloat16 pag_round(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half pag_round(float v) { return __float2half_rn(v); }


// Nearly always a division in 32 bits.  The long one is a call: its code in every place was fetched from memory by each
// launch (6 sequences behind 8192 shared positions: 30.6 -> 30.2 us).
static __device__ __noinline__ long long share_div_wide(long long a, long long b) { return a / b; }
__device__ __forceinline__ long long share_div(long long a, long long b) {
  return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : share_div_wide(a, b);
}

// Tiles of one warp's share: an equal part.  Where there are warps to spare a unit is cut into 128 pieces at most, of so
// many tiles that the partials (R rows of fp32) stay small beside the keys; and two units are not put on one warp either.
__device__ __forceinline__ long long tiles_per_worker(long long total, long long units, long long workers, int R) {
  const long long per = share_div(total + workers - 1, workers), unit = units > 0 ? share_div(total + units - 1, units) : 1;
  long long least = (unit + 127) / 128;
  if (least < (R > 16 ? R / 8 : 2)) least = R > 16 ? R / 8 : 2;
  if (least > unit) least = unit;
  return per < least ? least : per < 1 ? 1 : per;
}

// The line of `total` tiles shared out to all warps, those of the early CTAs first.  Early CTAs start beside the
// tensor-core tiles and get what they can do until those end on top of their equal share of the rest.
struct Shares {
  long long early, other;  // tiles per warp
  long long warps;         // of early CTAs
  __device__ __forceinline__ long long first_of(long long warp) const {
    return warp < warps ? warp * early : warps * early + (warp - warps) * other;
  }
  __device__ __forceinline__ long long warp_at(long long tile) const {
    const long long rest = tile - warps * early;
    return rest < 0 ? share_div(tile, early) : warps + share_div(rest, other);
  }
};
__device__ __forceinline__ Shares make_shares(const PagedAttParams& p, long long total, long long units, int warps_per_cta, int R) {
  const long long all = (long long)p.grid * warps_per_cta, early = (long long)p.early * warps_per_cta;
  const long long meanwhile = early * p.early_tiles;
  if (early == 0) return {0, tiles_per_worker(total, units, all, R), 0};
  if (total <= meanwhile) return {tiles_per_worker(total, units, early, R), 1, early};      // nothing is left for the others
  const long long other = share_div(total - meanwhile + all - 1, all);
  return {other + p.early_tiles, other, early};
}

// Positions [first, end) that the tensor-core unit of the stacked rows [row0, row0 + kTileRows) visits.
struct UnitKeys {
  int first, end;          // what some row of the unit sees
  int data_end;            // what the pages hold
};
__device__ __forceinline__ UnitKeys prefix_unit_keys(const PagedAttParams& p) { return UnitKeys{0, p.prefix, p.prefix}; }
// `rows`: how many of the unit's rows count (all of it, or its first tile)
__device__ __forceinline__ UnitKeys seq_unit_keys(const PagedAttParams& p, const SeqWork& w, int row0, int rows) {
  UnitKeys u{p.prefix, w.len, w.len};
  if (p.causal) {
    const int last = min(row0 + rows, w.n * p.G) - 1;
    u.end = min(w.len, w.len - w.n + last / p.G + 1);
  }
  return u;
}
// 128-key steps [a, b) of part s of `parts` of a unit's keys
__device__ __forceinline__ void unit_steps(const UnitKeys& u, int parts, int s, int& a, int& b) {
  const int j0 = u.first / kTileKeys, j1 = u.end > u.first ? (u.end + kTileKeys - 1) / kTileKeys : j0;
  const int64_t n = j1 - j0;
  a = j0 + (int)(n * s / parts);
  b = j0 + (int)(n * (s + 1) / parts);
}

// Whether a unit of `rows` rows shares its steps out between the two pipelines of a CTA: two partials a part.
__device__ __forceinline__ bool unit_is_dual(const PagedAttParams& p, bool of_sequence, int rows) {
  return rows <= kTileRows / 2 && (!of_sequence || p.seq_dual);
}

// paged_tile.cu: sets p.pre_tile, p.seq_tile and the splits by what the tensor-core tiles can and should take
// (tile_o / tile_ml are then wanted), and launches them.
void plan_paged_tiles(PagedAttParams& p, const arke_b200_paged_kv* d, int sms);
constexpr int kNoTiles = 1;   // nothing was launched: the caches' strides do not fit a tensor map
int launch_paged_tiles(const PagedAttParams& p, const arke_b200_paged_kv* d, cudaStream_t st);
// most partial rows ([2 * split][T * Hq], prefix and sequences) a plan can ask for
void paged_tile_rows(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t prefix, int sms, int64_t rows[2]);

}  // namespace arke
