// Attention over a paged cache on tcgen05 / TMEM / TMA, where many query rows read the same keys: the
// stacked rows of all sequences over a shared prefix, and the tokens of a prompt chunk.
//
// The pipeline is gqa_fwd_kernel's: two 128-row tiles per CTA, S = Q K^T (operands in shared memory), softmax in
// registers with one thread per row, P written over S in tensor memory in 16 bits, O += P V with P read from
// tensor memory, the running maximum moved only when it grows by 2^8.  What is different:
//   rows     row r of a unit is (token r / G, head r % G) of one key head: a TMA box of 128 / G tokens x G heads where
//            G divides 128, else every thread copies its own row of Q; each row has its own limit of visible keys;
//   keys     a 128-key tile is gathered page by page, one TMA box per page (128 / page_size boxes, or part of one
//            page), a lane of the loading warp each (one warp for K, one for V: with one for both, pages of 16 ran at
//            the pace of its instructions, 159 instead of 134 us for the chunk below); pages the sequence does not
//            have are loaded out of bounds, which fills zeros;
//   V        rows behind the sequence's end in its last page hold whatever memory held: 0 * NaN would reach O, so they
//            are zeroed in shared memory before the product (the first tile, and the one in which the data ends);
//   split    a unit's keys are shared out over `split` CTAs, and the (m, l, O) partials meet in the join kernel;
//   dual     a unit of at most 128 rows has one query tile, whose steps the two pipelines take in turn.
//
// Bound: the softmax arithmetic per SM (about 2900 cycles per 128-key step of two tiles, against 2048 of tensor
// core work), as in gqa_fwd_kernel; a step streams 64 KB, at that pace 22 B per clock and SM, just the HBM rate.
// Measured 1.7 us a step (tensor pipe 56 % active) and about 10 us a CTA for its start and end.  Two chunks of 512
// tokens over 8192 positions (32 / 8 heads, D = 128, 133 GFLOP): 135 us, 0.99 PFLOP/s on 128 of 148 SMs.  A shared
// prefix beside streamed keys of the sequences' own: see plan_paged_tiles.
#include "paged_att.cuh"
#include <math.h>

namespace arke {

constexpr int kTileThreads = 384;      // 3 warpgroups: softmax tile 0, softmax tile 1, {K loads, MMA, V repair, V loads}
constexpr float kTileRescale = 8.f;    // log2 units

template <int D>
struct TileSmem {
  static constexpr int kChunks = D / 64;                     // 64-element (128-byte) chunks per row
  static constexpr int kTileBytes = 128 * D * 2;
  static constexpr int kChunkBytes = 128 * 128;
  static constexpr int kQOff = 0;                            // Q0, Q1
  static constexpr int kKOff = 2 * kTileBytes;               // K stage 0, 1
  static constexpr int kVOff = 4 * kTileBytes;               // V stage 0, 1
  static constexpr int kBarOff = 6 * kTileBytes;
  static constexpr int kNumBars = 20;
  static constexpr int kMiscOff = kBarOff + kNumBars * 8;
  static constexpr int kTotal = kMiscOff + 64 + 1024;        // + alignment slack
};

__device__ __forceinline__ bool tile_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitLimitCycles) return false;
  }
  return true;
}
__device__ __forceinline__ void tile_abort(int* status, volatile int* abort_flag, int code) {
  atomicCAS(status, 0, code);
  *abort_flag = 1;
  __threadfence_block();
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

struct TileGeometry {
  int pre_pairs;       // row-tile pairs of the prefix, 0: none
  int box_rows;        // rows of a TMA box: min(page_size, 128)
  int k_order, v_order;   // dimensions 1 to 3 of the tensor maps, 2 bits each, in the order of their strides: 0 row, 1 head, 2 page
  int q_tma;           // Q tiles are boxes of 128 / G tokens x G heads
};

template <int D, bool IS_BF16>
__global__ void __launch_bounds__(kTileThreads, 1)
paged_tile_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const PagedAttParams p, const TileGeometry geo) {
  using SM = TileSmem<D>;
  constexpr int KSTEPS_QK = D / 16;
  constexpr int KSTEPS_PV = kTileKeys / 16;
  constexpr uint32_t TMEM_COLS = 512;
  constexpr uint32_t S_COL0 = 0, S_COL1 = 128, O_COL0 = 256, O_COL1 = 256 + D;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ int s_scan[kTileThreads / 32];
  __shared__ int s_find[2];
  pdl_launch_dependents();             // the streaming kernel needs nothing from this one until it ends
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- which unit, which part of its keys
  int idx = blockIdx.x;
  const int pre_ctas = geo.pre_pairs * p.kv.Hkv * p.pre_split;
  const int tokens = seq_begin_clamped(p.kv, p.kv.B);
  int b = -1, pair, h, part, parts;
  SeqWork w{tokens, p.prefix, 0};
  UnitKeys keys;
  int tok0 = 0;
  if (idx < pre_ctas) {
    parts = p.pre_split;
    part = idx % parts;
    h = idx / parts % p.kv.Hkv;
    pair = idx / (parts * p.kv.Hkv);
    keys = prefix_unit_keys(p);
  } else {
    idx -= pre_ctas;
    parts = p.seq_split;
    part = idx % parts;
    h = idx / parts % p.kv.Hkv;
    const int want = idx / (parts * p.kv.Hkv);           // number of the pair among those of all sequences
    int base = 0;
    if (threadIdx.x == 0) s_find[0] = -1;
    for (int b0 = 0; b0 < p.kv.B; b0 += kTileThreads) {
      const int bb = b0 + threadIdx.x;
      int n = 0;
      if (bb < p.kv.B) {
        const SeqWork o = seq_work(p, bb);
        if (seq_in_tiles(p, o.n)) n = (o.n * p.G + kTileRows - 1) / kTileRows;
      }
      int inc = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += v;
      }
      if (lane == 31) s_scan[warp] = inc;
      __syncthreads();
      int end = base + inc, sum = 0;
      for (int i = 0; i < kTileThreads / 32; ++i) {
        if (i < warp) end += s_scan[i];
        sum += s_scan[i];
      }
      if (end - n <= want && want < end) { s_find[0] = bb; s_find[1] = want - (end - n); }
      base += sum;
      __syncthreads();
      if (base > want) break;
    }
    __syncthreads();
    b = s_find[0];
    if (b < 0) return;
    pair = s_find[1];
    w = seq_work(p, b);
    tok0 = seq_begin_clamped(p.kv, b);
    keys = seq_unit_keys(p, w, pair * kTileRows, kTileRows);
  }
  const int row0 = pair * kTileRows;
  const int rows = min(kTileRows, w.n * p.G - row0);
  int j0, j1;
  unit_steps(keys, parts, part, j0, j1);
  if (rows <= 0 || j0 >= j1) return;                     // nothing to see: the join knows
  // Steps of each tile.  A unit of at most 128 rows has one query tile: the two pipelines then take its even and odd
  // steps and leave a partial each, instead of one waiting for the other's softmax.  Else a causal chunk's first rows
  // see fewer keys than its last.
  const int steps = j1 - j0;
  const bool dual = unit_is_dual(p, b >= 0, rows);
  int n0 = steps, n1 = steps;
  if (dual) {
    n0 = (steps + 1) >> 1;
    n1 = steps >> 1;
  } else {
    if (rows <= 128) n1 = 0;
    if (b >= 0) {
      const UnitKeys k0 = seq_unit_keys(p, w, row0, 128);
      n0 = max(0, min(j1, (k0.end + kTileKeys - 1) / kTileKeys) - j0);
    }
  }
  const bool fix_first = j0 * kTileKeys < keys.first;    // V rows that are not this unit's

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::kBarOff);
  uint64_t* q_full = bars;          // [2]
  uint64_t* k_full = bars + 2;      // [2]
  uint64_t* k_empty = bars + 4;     // [2]
  uint64_t* v_full = bars + 6;      // [2]
  uint64_t* v_empty = bars + 8;     // [2]
  uint64_t* s_full = bars + 10;     // [2] per query tile
  uint64_t* p_ready = bars + 12;    // [2] per query tile
  uint64_t* pv_done = bars + 14;    // [2] per query tile
  uint64_t* p_half = bars + 16;     // [2] per query tile: first 64 keys of P are in tensor memory
  uint64_t* v_fix = bars + 18;      // [2] V rows in front of the unit's keys are zero; V of the tile in which the data ends has arrived
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::kMiscOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + SM::kMiscOff + 4);
  volatile int* bad_flag = reinterpret_cast<volatile int*>(smem + SM::kMiscOff + 8);

  if (threadIdx.x == 0) {
    mbar_init(&q_full[0], geo.q_tma ? 1 : 128);
    mbar_init(&q_full[1], geo.q_tma ? 1 : 128);
    for (int i = 2; i < 12; ++i) mbar_init(&bars[i], 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&p_ready[t], 4);   // one arrival per softmax warp (lane 0 after __syncwarp)
      mbar_init(&pv_done[t], 1);
      mbar_init(&p_half[t], 4);
    }
    mbar_init(&v_fix[0], 1);
    mbar_init(&v_fix[1], 1);
    *abort_flag = 0;
    *bad_flag = 0;
    fence_mbar_init();
    if (geo.q_tma) tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  // Zeroes the V rows of step j outside [first, data_end), which `full` says are there, and reports that to `done`.
  auto repair = [&](int j, int data_end, uint64_t* full, uint64_t* done) -> bool {
    const bool got = tile_wait(full, 0, abort_flag);
    if (!__all_sync(0xffffffffu, got)) return false;
    const int k0 = (j0 + j) * kTileKeys;
    uint8_t* v = smem + SM::kVOff + (j & 1) * SM::kTileBytes;
    for (int r = lane; r < kTileKeys; r += 32) {
      if (k0 + r >= keys.first && k0 + r < data_end) continue;
#pragma unroll
      for (int c = 0; c < SM::kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(v + c * SM::kChunkBytes + r * 128 + i * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(done);
    return true;
  };

  if (warp >= 8) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
   if (warp == 8 || warp == 11) {
    // =============================== TMA producers: K (warp 8), V (warp 11) ===============================
    // lane i owns the box of keys [i * box_rows, (i + 1) * box_rows) of every tile
    const bool is_k = warp == 8;
    const int boxes = kTileKeys / geo.box_rows;
    const CUtensorMap* map = is_k ? &tmap_k : &tmap_v;
    const int order = is_k ? geo.k_order : geo.v_order;
    auto pick = [&](int d, int row, int page) {
      const int which = (order >> (2 * d)) & 3;
      return which == 0 ? row : which == 1 ? h : page;
    };
    uint64_t* full = is_k ? k_full : v_full;
    uint64_t* empty = is_k ? k_empty : v_empty;
    uint8_t* dst = smem + (is_k ? SM::kKOff : SM::kVOff) + lane * geo.box_rows * 128;
    const int data_end = b < 0 ? prefix_data_end(p) : keys.data_end;
    // the step inside which the data ends, -1 where none does
    const int fix_step = data_end % kTileKeys != 0 && data_end / kTileKeys >= j0 && data_end / kTileKeys < j1 ? data_end / kTileKeys - j0 : -1;
    auto lookup = [&](int step) -> int {                 // physical page, num_pages (out of bounds) where there is none
      const int key = (j0 + step) * kTileKeys + lane * geo.box_rows;
      if (lane >= boxes || step >= steps || key >= data_end || key + geo.box_rows <= keys.first) return p.kv.num_pages;
      const int id = page_of(p, b, key / p.kv.page_size);
      if (id >= 0 && id < p.kv.num_pages) return id;
      *bad_flag = 1;
      atomicCAS(p.status, 0, KSTAT_BAD_INDEX);
      return p.kv.num_pages;
    };
    int page = lookup(0);
    bool ok = true;
    if (is_k && geo.q_tma && lane < 2 && (lane ? n1 : n0) > 0) {   // lane t: query tile t (128 rows are whole tokens)
      mbar_arrive_expect_tx(&q_full[lane], SM::kTileBytes);
#pragma unroll
      for (int c = 0; c < SM::kChunks; ++c)
        tma_load_3d(smem + SM::kQOff + lane * SM::kTileBytes + c * SM::kChunkBytes, &tmap_q, &q_full[lane], c * 64, h * p.G,
                    tok0 + (row0 + (dual ? 0 : lane * 128)) / p.G);
    }
    for (int j = 0; j < steps; ++j) {
      const int s = j & 1;
      const int next = lookup(j + 1);
      ok = tile_wait(&empty[s], ((j >> 1) & 1) ^ 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      // V of that step arrives at a barrier of its own, and the stage is full when its rows behind the end are zero
      const bool fix = !is_k && j == fix_step;
      uint64_t* arrived = fix ? &v_fix[1] : &full[s];
      if (lane == 0) mbar_arrive_expect_tx(arrived, SM::kTileBytes);
      __syncwarp();
      if (lane < boxes) {
        const int row = ((j0 + j) * kTileKeys + lane * geo.box_rows) % p.kv.page_size;
#pragma unroll
        for (int c = 0; c < SM::kChunks; ++c)
          tma_load_4d(dst + s * SM::kTileBytes + c * SM::kChunkBytes, map, arrived, c * 64, pick(0, row, page), pick(1, row, page),
                      pick(2, row, page));
      }
      page = next;
      if (fix && !repair(j, data_end, arrived, &full[s])) { ok = false; break; }
    }
    if (!ok && lane == 0) tile_abort(p.status, abort_flag, KSTAT_TIMEOUT_PRODUCER);
   } else if (warp == 9) {
    // =============================== MMA issuer ===============================
    if (elect_one()) {
      const uint32_t fmt = IS_BF16 ? UMMA_BF16 : UMMA_F16;
      const uint32_t idesc_qk = make_idesc(UMMA_C_F32, fmt, fmt, 0, 0, 128, kTileKeys);
      const uint32_t idesc_pv = make_idesc(UMMA_C_F32, fmt, fmt, 0, 1, 128, D);
      const uint32_t hi_k = smem_desc_hi_sw128(1024);
      const uint32_t q_lo0 = smem_desc_lo(smem_u32(smem + SM::kQOff), 16), k_lo0 = smem_desc_lo(smem_u32(smem + SM::kKOff), 16);
      const uint32_t v_lo0 = smem_desc_lo(smem_u32(smem + SM::kVOff), SM::kChunkBytes);
      constexpr uint32_t kTileLo = SM::kTileBytes >> 4;
      bool ok = true;

      auto issue_qk = [&](int t, int step) -> bool {  // S_t = Q_t K_step^T
        const int st = step & 1;
        if (!tile_wait(&k_full[st], (step >> 1) & 1, abort_flag)) return false;
        tc_fence_after();
        const uint32_t qa = q_lo0 + t * kTileLo;
        const uint32_t ka = k_lo0 + st * kTileLo;
        const uint32_t d = tmem_base + t * S_COL1;
#pragma unroll
        for (int k = 0; k < KSTEPS_QK; ++k) {
          const uint32_t off = ((k >> 2) * SM::kChunkBytes + (k & 3) * 32) >> 4;
          if (k == 0) umma_ss_f16_lohi<false>(d, qa + off, hi_k, ka + off, hi_k, idesc_qk);
          else umma_ss_f16_lohi<true>(d, qa + off, hi_k, ka + off, hi_k, idesc_qk);
        }
        tc_commit(&s_full[t]);
        return true;
      };
      // O_t (+)= P_t V_step in two halves of 64 keys; i: how many steps this tile had before
      auto issue_pv = [&](int t, int i, int step) -> bool {
        const int st = step & 1;
        if (!tile_wait(&p_half[t], i & 1, abort_flag) || !tile_wait(&v_full[st], (step >> 1) & 1, abort_flag)) return false;
        if (step == 0 && fix_first && !tile_wait(&v_fix[0], 0, abort_flag)) return false;
        tc_fence_after();
        const uint32_t va = v_lo0 + st * kTileLo;
        const uint32_t d = tmem_base + O_COL0 + t * D;
        const uint32_t pa = tmem_base + t * S_COL1;
        if (i == 0) umma_ts_f16_lohi<false>(d, pa, va, hi_k, idesc_pv);
        else umma_ts_f16_lohi<true>(d, pa, va, hi_k, idesc_pv);
#pragma unroll
        for (int kk = 1; kk < KSTEPS_PV / 2; ++kk) umma_ts_f16_lohi<true>(d, pa + kk * 8, va + kk * (2048 >> 4), hi_k, idesc_pv);
        if (!tile_wait(&p_ready[t], i & 1, abort_flag)) return false;
        tc_fence_after();
#pragma unroll
        for (int kk = KSTEPS_PV / 2; kk < KSTEPS_PV; ++kk) umma_ts_f16_lohi<true>(d, pa + kk * 8, va + kk * (2048 >> 4), hi_k, idesc_pv);
        tc_commit(&pv_done[t]);
        return true;
      };

      // A stage is free after the last product that reads it: the only one's where the tiles take turns (dual), else
      // tile 1's, or tile 0's where tile 1 has no such step.
      if (n0 > 0) ok = tile_wait(&q_full[0], 0, abort_flag) && issue_qk(0, 0);
      if (ok && dual) tc_commit(&k_empty[0]);
      if (ok && n1 > 0) ok = tile_wait(&q_full[1], 0, abort_flag) && issue_qk(1, dual ? 1 : 0);
      if (ok && (!dual || n1 > 0)) tc_commit(&k_empty[dual ? 1 : 0]);
      const int n_max = max(n0, n1);
#pragma unroll 1
      for (int i = 0; i < n_max && ok; ++i) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int n_t = t ? n1 : n0;
          if (i >= n_t) continue;
          const int step = dual ? 2 * i + t : i, next = step + (dual ? 2 : 1);
          if (!issue_pv(t, i, step)) { ok = false; break; }
          if (dual || t == 1 || i >= n1) tc_commit(&v_empty[step & 1]);
          if (i + 1 < n_t && !issue_qk(t, next)) { ok = false; break; }
          if (dual && i + 1 < n_t) tc_commit(&k_empty[next & 1]);
        }
        if (ok && !dual && i + 1 < n_max) tc_commit(&k_empty[(i + 1) & 1]);
      }
      if (!ok) tile_abort(p.status, abort_flag, KSTAT_TIMEOUT_MMA);
    }
   } else if (warp == 10 && fix_first) {
    // the first tile's V: stage 0 cannot move on before this is done
    if (!repair(0, keys.data_end, &v_full[0], &v_fix[0]) && lane == 0) tile_abort(p.status, abort_flag, KSTAT_TIMEOUT_PRODUCER);
   }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // ===================== softmax / correction / epilogue warps =====================
    const int t = warp >> 2;                     // query tile handled by this warpgroup
    const int quarter = warp & 3;                // TMEM lane quarter this warp may touch
    const int row_in_tile = quarter * 32 + lane;
    const int in_unit = (dual ? 0 : t * 128) + row_in_tile;
    const int rr = row0 + in_unit;               // stacked row
    const bool row_ok = in_unit < rows;
    const int n_t = t ? n1 : n0;
    const int token = tok0 + (row_ok ? rr / p.G : 0), head = h * p.G + (row_ok ? rr % p.G : 0);

    // ---- this thread's row of Q, in the layout the tensor core reads (128-byte rows, 16-byte chunks swizzled)
    if (n_t > 0 && !geo.q_tma) {
      uint8_t* dst = smem + SM::kQOff + t * SM::kTileBytes + row_in_tile * 128;
      const int64_t at = token * p.q_st + head * p.q_sh;
      const bool copy = row_ok && q_chk(p, at, D);
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.q) + at);
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint4 v = copy ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + (i >> 3) * SM::kChunkBytes + (((i & 7) ^ (row_in_tile & 7)) << 4)) = v;
      }
      fence_async_smem();
      mbar_arrive(&q_full[t]);
    }
    // ---- last position this row sees among the unit's keys (rows not in use: all, so that they ask for no mask)
    int limit = 0x7fffffff;
    if (b >= 0) {
      if (row_ok) limit = (p.causal ? w.len - w.n + (token - tok0) + 1 : w.len) - 1;
    } else {
      const int t_last = (row0 + rows - 1) / p.G;        // lanes without a row search for the last one's
      const int seen = seen_by(p, find_sequence_lanes(p.kv, row_ok ? token : t_last), token);
      if (row_ok) limit = min(seen, p.prefix) - 1;
    }
    const int warp_limit = __reduce_min_sync(0xffffffffu, limit);

    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_off + (t == 0 ? S_COL0 : S_COL1);
    const uint32_t o_addr = tmem_base + lane_off + (t == 0 ? O_COL0 : O_COL1);
    const float c = p.scale_log2;
    float m_used = -INFINITY;   // running max (log2 domain, scale included) the sums are based on
    float l = 0.f;              // running sum of 2^(s - m_used)
    bool ok = true;

    for (int j = 0; j < n_t; ++j) {
      const uint32_t jp = j & 1;
      bool got = tile_wait(&s_full[t], jp, abort_flag);
      if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
      tc_fence_after();
      const int k0 = (j0 + (dual ? 2 * j + t : j)) * kTileKeys;
      const bool need_mask = k0 < keys.first || k0 + kTileKeys - 1 > warp_limit;
      uint32_t v[4][32];
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) tmem_ld32(s_addr + ch * 32, v[ch]);
      tmem_ld_wait();
      if (need_mask) {
#pragma unroll
        for (int ch = 0; ch < 4; ++ch)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (k0 + ch * 32 + i > limit || k0 + ch * 32 + i < keys.first) v[ch][i] = 0xff800000u;  // -inf
      }
      float mc[16];
#pragma unroll
      for (int ch = 0; ch < 4; ++ch)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
          const int b0 = q4 * 8;
          float a = max3(__uint_as_float(v[ch][b0]), __uint_as_float(v[ch][b0 + 1]), __uint_as_float(v[ch][b0 + 2]));
          a = max3(a, __uint_as_float(v[ch][b0 + 3]), __uint_as_float(v[ch][b0 + 4]));
          a = max3(a, __uint_as_float(v[ch][b0 + 5]), __uint_as_float(v[ch][b0 + 6]));
          mc[ch * 4 + q4] = fmaxf(a, __uint_as_float(v[ch][b0 + 7]));
        }
#pragma unroll
      for (int i = 0; i < 5; ++i) mc[i] = max3(mc[i], mc[5 + 2 * i], mc[6 + 2 * i]);
      mc[0] = max3(mc[0], mc[1], mc[2]);
      const float mx = max3(mc[0], mc[3], fmaxf(mc[4], mc[15]));
      const float m_new = fmaxf(m_used, mx * c);
      const bool want = (j > 0) && (m_new > m_used + kTileRescale);
      if (j == 0) {
        m_used = m_new;
      } else if (__any_sync(0xffffffffu, want)) {
        got = tile_wait(&pv_done[t], (j - 1) & 1, abort_flag);
        if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
        tc_fence_after();
        const float alpha = m_new == m_used ? 1.f : ex2_approx(m_used - m_new);   // both may be -inf still
#pragma unroll 1
        for (int ch = 0; ch < D / 32; ++ch) {
          uint32_t o[32];
          tmem_ld32(o_addr + ch * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st32(o_addr + ch * 32, o);
        }
        tmem_st_wait();
        l *= alpha;
        m_used = m_new;
      }
      const float shift = m_used == -INFINITY ? 0.f : -m_used;    // a row that has seen nothing yet: 2^(-inf) = 0
      const uint64_t c2 = f2_pack(c, c);
      const uint64_t nm2 = f2_pack(shift, shift);
      uint64_t sum2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint64_t tt = f2_fma(f2_pack(__uint_as_float(v[ch][2 * i]), __uint_as_float(v[ch][2 * i + 1])), c2, nm2);
          float t0, t1;
          f2_unpack(tt, t0, t1);
          const float p0 = ex2_approx(t0), p1 = ex2_approx(t1);
          sum2[i & 3] = f2_add(sum2[i & 3], f2_pack(p0, p1));
          // P in 16 bits is what the tensor core multiplies: off by half a step each, like the result's own rounding
          pk[i] = IS_BF16 ? pack_bf16x2(p0, p1) : pack_f16x2(p0, p1);
        }
        tmem_st16(s_addr + ch * 16, pk);
        if (ch == 1) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_half[t]);
        }
      }
      {
        float a0, a1;
        f2_unpack(f2_add(f2_add(sum2[0], sum2[1]), f2_add(sum2[2], sum2[3])), a0, a1);
        l += a0 + a1;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[t]);
    }

    // ---- epilogue: the finished rows, or this part's (m, l, O) ----
    if (ok && n_t > 0) {
      const bool got = tile_wait(&pv_done[t], (n_t - 1) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, got)) ok = false;
    }
    if (ok && (n_t > 0 || !dual)) {                      // a pipeline without steps leaves no partial
      tc_fence_after();
      const int64_t all = (int64_t)p.kv.T * p.Hq;
      const int orow = row_ok ? token * p.Hq + head : -1;
      const bool final_here = b >= 0 && !dual && p.seq_split == 1 && p.prefix == 0;
      const int slot = dual ? 2 * part + t : part;
      [[maybe_unused]] const int64_t out_row = final_here ? orow : slot * all + orow, out_rows = final_here ? all : p.tile_rows[b >= 0];
      const bool write = orow >= 0 && ARKE_CHK(orow, orow, all) && ARKE_CHK(out_row, out_row, out_rows);
      const unsigned live = __ballot_sync(0xffffffffu, write);
      // a missing page, or nothing seen (NaN scores leave a sum): O is not what tensor memory holds
      const bool broken = *bad_flag != 0, none = broken || m_used == -INFINITY;
      const float fill = broken || l != 0.f ? __uint_as_float(0x7fc00000u) : 0.f;
      if (broken) { l = fill; m_used = 0.f; }
      const float scale = !final_here ? 1.f : l == 0.f ? 0.f : 1.f / l;
      // Rows leave through shared memory (Q's, which no MMA reads any more), so that a warp's stores are whole lines
      // and not 32 pieces of 16 bytes: 32 columns of 32 rows a turn, 16-byte chunks swizzled by the row.
      uint8_t* stage = smem + SM::kQOff + t * SM::kTileBytes + quarter * 32 * 128;
      uint8_t* base = final_here ? reinterpret_cast<uint8_t*>(p.o) : reinterpret_cast<uint8_t*>(p.tile_o[b >= 0] + slot * all * D);
#pragma unroll 1
      for (int ch = 0; ch < D / 32 && live != 0; ++ch) {
        uint32_t o[32];
        if (n_t > 0) {
          tmem_ld32(o_addr + ch * 32, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(none ? fill : __uint_as_float(o[i]) * scale);
        if (final_here) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            o[i] = IS_BF16 ? pack_bf16x2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]))
                           : pack_f16x2(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < 4 || !final_here)
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((i ^ (lane & 7)) << 4)) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        __syncwarp();
        const int chunks = final_here ? 4 : 8, log_chunks = final_here ? 2 : 3, row_bytes = D * chunks / 2;
#pragma unroll 4
        for (int i = lane; i < 32 * chunks; i += 32) {
          const int r = i >> log_chunks, c = i & (chunks - 1);
          const int64_t to = __shfl_sync(0xffffffffu, orow, r);
          if ((live >> r) & 1)
            *reinterpret_cast<uint4*>(base + to * row_bytes + (ch * chunks + c) * 16) = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
        }
        __syncwarp();
      }
      if (write && !final_here) *reinterpret_cast<float2*>(p.tile_ml[b >= 0] + (slot * all + orow) * 2) = make_float2(m_used, l);
      if (write && final_here && p.lse) p.lse[orow] = l == 0.f ? -INFINITY : (m_used + log2f(l)) * 0.6931471805599453f;
    } else if (!ok && lane == 0) {
      tile_abort(p.status, abort_flag, KSTAT_TIMEOUT_SOFTMAX);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    if (*abort_flag) {
      const long long t0 = clock64();
      while (clock64() - t0 < 2000000LL) { __nanosleep(1000); }
    }
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------------------- host
static int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// CTAs that share a unit's keys: as many as fill the SMs once
static int tile_split(int64_t units, int sms) {
  const int64_t s = units > 0 ? sms / units : 1;
  return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
}
// but no more than leave each at least four 128-key steps: a part costs about as much as that before its first step
// and after its last one, and its partial rows have to be joined
static int useful_split(int split, int64_t keys) {
  const int64_t most = keys / (4 * kTileKeys);
  return most < 1 ? 1 : most < split ? (int)most : split;
}

// Units that T tokens of B sequences make, at most: one for every 256 rows and one more for each sequence's rest.
static int64_t tile_units(int64_t T, int64_t B, int64_t G, int64_t Hkv, bool prefix) {
  const int64_t rows = T * G, rests = B < rows / (kFewRows + 1) ? B : rows / (kFewRows + 1);
  return (prefix ? div_up(rows, kTileRows) : rows / kTileRows + (rests > 0 ? rests : 1)) * Hkv;
}
// Sequences' units of one query tile use both pipelines where partials are wanted anyway, or most units are such.
static bool seq_units_dual(int64_t T, int64_t B, int64_t G, int64_t prefix, int split) {
  return prefix > 0 || split > 1 || T * G <= B * (kTileRows / 2);
}

void paged_tile_rows(int64_t T, int64_t B, int64_t Hq, int64_t Hkv, int64_t prefix, int sms, int64_t rows[2]) {
  rows[0] = rows[1] = 0;
  const int64_t G = Hq / Hkv;
  if (T * G <= kFewPrefixRows) return;
  if (prefix > 0) rows[0] = 2 * T * Hq * tile_split(tile_units(T, B, G, Hkv, true), sms);
  const int split = tile_split(tile_units(T, B, G, Hkv, false), sms);
  if (seq_units_dual(T, B, G, prefix, split)) rows[1] = 2 * T * Hq * split;
}

void plan_paged_tiles(PagedAttParams& p, const arke_b200_paged_kv* d, int sms) {
  p.pre_tile = p.seq_tile = 0;
  p.pre_split = p.seq_split = 1;
  p.seq_dual = p.early = p.early_tiles = 0;
  const int64_t page = d->page_size, rows = (int64_t)p.kv.T * p.G;
  // A tile is put together from whole pages (or lies in one) in 8-row groups, the unit of the swizzle; Q rows are
  // copied 16 bytes at a time.  Anything else stays with the streaming kernel.
  const bool pages_ok = (page % 8 == 0 && kTileKeys % page == 0) || page % kTileKeys == 0;
  const bool q_ok = (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && p.q_st % 8 == 0 && p.q_sh % 8 == 0;
  if (!pages_ok || !q_ok || d->num_pages == 0 || p.kv.B == 0 || rows <= kFewPrefixRows) return;
  p.pre_tile = p.prefix >= kTileKeys;
  // Without cu_q every sequence has the same tokens.  With it only the caller can know the longest's.  Unknown, one may
  // have T - B + 1 where every sequence has a token, and the launch pays when that could fill a unit; a longer one among
  // empty slots then stays with the streaming kernel, whose blocks of at most kFewRows rows read the keys again each
  // (512 tokens over 4096 positions beside 511 empty slots, 32 / 8 heads, D = 128: 606 us unknown, 76 us told, 58 us
  // without the slots).  Taking T for granted would put a launch of idle tiles in front of every decode batch.
  p.seq_tile = !p.kv.cu ? (int64_t)p.kv.uniform * p.G > kFewRows
               : p.kv.max_new ? (int64_t)(p.kv.max_new < p.kv.T ? p.kv.max_new : p.kv.T) * p.G > kFewRows
                              : (int64_t)(p.kv.T - p.kv.B + 1) * p.G > kTileRows;
  const int64_t G = p.G;
  if (p.pre_tile) {
    const int64_t units = tile_units(p.kv.T, p.kv.B, G, p.kv.Hkv, true);
    p.pre_split = useful_split(tile_split(units, sms), p.prefix);
    // The tiles are bound by arithmetic and the sequences' own keys by HBM: side by side, on SMs of their own, they take
    // less than one after the other.  Tiles get three quarters of the SMs, or half where the keys then do not fit beside
    // them.  How many keys follow only the device knows: the guess is half of what the table has room for, at 13 GB/s a
    // streaming CTA.  Measured in us, tiles on all SMs / on 3/4 / on 1/2 (32 / 8 heads, D = 128):
    //   6 of <= 700 keys behind 8192: 32 / 24 / 25       8 of <= 1500 behind 16384: 47 / 32 / 34
    //   128 of <= 64 behind 16384: 63 / 59 / 75          128 of <= 512 behind 16384: 93 / 90 / 77
    //   64 of <= 600 behind 8192: 56 / - / 46            16 of <= 3000 behind 18432: 61 / - / 44
    const double own = (double)((int64_t)p.kv.max_pages * p.kv.page_size - p.prefix) * p.kv.B * p.kv.Hkv * d->head_dim * 4;
    const int steps = (p.prefix + kTileKeys - 1) / kTileKeys;
    for (int part = 3; part >= 2 && !p.seq_tile && own > 0; --part) {
      const int64_t fewer = sms * part / 4 / units;
      if (fewer >= 1 && fewer < p.pre_split) p.pre_split = (int)fewer;
      const int64_t left = sms - units * p.pre_split;
      if (left < 16) break;
      p.early = 2 * (int)left;
      const double us = 10.0 + 1.7 * steps / p.pre_split;        // the tiles' time
      // 0.9 tiles of 8 KB a microsecond and warp (with 0.6: 0 to 11 % slower, with 1.2: 0 to 7 %)
      p.early_tiles = (int)(0.9 * us);
      if (own <= 26e3 * p.early * us) break;
    }
  }
  if (p.seq_tile) {
    const int split = tile_split(tile_units(p.kv.T, p.kv.B, G, p.kv.Hkv, false), sms);
    p.seq_split = useful_split(split, (int64_t)p.kv.max_pages * p.kv.page_size - p.prefix);
    p.seq_dual = seq_units_dual(p.kv.T, p.kv.B, G, p.prefix, split);
  }
}

// K or V as a tensor {D, then page row, head and page in the order of their strides}
static int page_map(CUtensorMap* m, const void* base, int64_t sp, int64_t sh, int64_t sr, const arke_b200_paged_kv* d, int box_rows,
                    int* order) {
  const int64_t stride[3] = {sr, sh, sp}, extent[3] = {d->page_size, d->heads, d->num_pages};
  int at[3] = {0, 1, 2};
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 2; ++j)
      if (stride[at[j]] > stride[at[j + 1]]) { const int t = at[j]; at[j] = at[j + 1]; at[j + 1] = t; }
  uint64_t dims[4] = {(uint64_t)d->head_dim}, str[3];
  uint32_t box[4] = {64};
  *order = 0;
  for (int i = 0; i < 3; ++i) {
    dims[i + 1] = (uint64_t)extent[at[i]];
    // a dimension of one has no stride worth the name
    str[i] = (uint64_t)(extent[at[i]] == 1 && stride[at[i]] == 0 ? d->head_dim : stride[at[i]]) * 2;
    box[i + 1] = at[i] == 0 ? (uint32_t)box_rows : 1u;
    *order |= at[i] << (2 * i);
  }
  return make_tensor_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, base, dims, str, box, 1, "paged_gqa_fwd");
}

template <int D, bool IS_BF16>
static int launch_tiles(const PagedAttParams& p, const arke_b200_paged_kv* d, cudaStream_t st) {
  using SM = TileSmem<D>;
  TileGeometry geo{};
  geo.box_rows = (int)(d->page_size < kTileKeys ? d->page_size : kTileKeys);
  CUtensorMap tq{}, tk, tv;
  int rc = ARKE_OK;
  geo.q_tma = 128 % p.G == 0 && p.q_sh * p.Hq <= p.q_st;     // heads inside their token's row: strides in ascending order
  if (geo.q_tma) {
    uint64_t dims[3] = {(uint64_t)D, (uint64_t)p.Hq, (uint64_t)p.kv.T};
    uint64_t str[2] = {(uint64_t)p.q_sh * 2, (uint64_t)p.q_st * 2};
    uint32_t box[3] = {64, (uint32_t)p.G, (uint32_t)(128 / p.G)};
    if (make_tensor_map(&tq, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, p.q, dims, str, box, 1, "paged_gqa_fwd") != ARKE_OK) geo.q_tma = 0;
  }
  rc = page_map(&tk, d->k, p.kv.ksp, p.kv.ksh, p.kv.ksr, d, geo.box_rows, &geo.k_order);
  if (rc == ARKE_OK) rc = page_map(&tv, d->v, p.kv.vsp, p.kv.vsh, p.kv.vsr, d, geo.box_rows, &geo.v_order);
  if (rc != ARKE_OK) return kNoTiles;                  // strides that no tensor map takes: the streaming kernel's
  const int64_t rows = (int64_t)p.kv.T * p.G;
  int64_t ctas = 0;
  if (p.pre_tile) {
    geo.pre_pairs = (int)div_up(rows, kTileRows);
    ctas += (int64_t)geo.pre_pairs * p.kv.Hkv * p.pre_split;
  }
  if (p.seq_tile) {
    // pairs of all sequences that qualify: one for every 256 rows and one more for each such sequence's rest
    int64_t pairs;
    if (!p.kv.cu) pairs = (int64_t)p.kv.B * div_up((int64_t)p.kv.uniform * p.G, kTileRows);
    else pairs = rows / kTileRows + (p.kv.B < rows / (kFewRows + 1) ? p.kv.B : rows / (kFewRows + 1));
    ctas += pairs * p.kv.Hkv * p.seq_split;
  }
  if (ctas > 0x7fffffffLL) return set_error(ARKE_ERR_SHAPE, "paged_gqa_fwd: too many query rows");
  auto kern = paged_tile_kernel<D, IS_BF16>;
  cudaError_t e = ensure_dynamic_smem(kern, SM::kTotal);
  if (e != cudaSuccess) return set_cuda_error("paged_gqa_fwd shared memory", e);
  kern<<<(unsigned)ctas, kTileThreads, SM::kTotal, st>>>(tq, tk, tv, p, geo);
  e = cudaGetLastError();
  return e == cudaSuccess ? ARKE_OK : set_cuda_error("paged_gqa_fwd tile launch", e);
}

int launch_paged_tiles(const PagedAttParams& p, const arke_b200_paged_kv* d, cudaStream_t st) {
  ARKE_CHK_BIND();
  if (d->dtype == ARKE_BF16) return d->head_dim == 128 ? launch_tiles<128, true>(p, d, st) : launch_tiles<64, true>(p, d, st);
  return d->head_dim == 128 ? launch_tiles<128, false>(p, d, st) : launch_tiles<64, false>(p, d, st);
}

}  // namespace arke
