// dc_weights.cu -- the softmax weight that every cached key receives.
//
//   acc[b][g][j] = decay acc[b][g][j] + sum over rows r and heads h of group g of exp(scale q_rh . k_j - lse_rh)
//
// With lse known the sum needs no running maximum and no second pass.  The
// product is formed as K Q^T: keys on the 128 TMEM lanes, up to 128 query rows
// (row, head of the group; heads innermost) on the columns.  A thread then holds
// one key against all rows (many: two threads, half of the columns each, joined at
// the end) and adds its exponentials in a register: no atomics, one order of
// summation.
//
// k_weights_few, up to 128 columns: a block keeps Q in shared memory and streams
// its share of the cache's keys (16 KB panels through a ring by TMA), two blocks an
// SM, scores double-buffered in TMEM.  HBM-bound: each key is read once.  The shares
// are of the cache's size, since the lengths are known on the device alone: 16
// sequences of 8 heads and 8192 keys take 49 us (5.6 TB/s) where all are full and 44
// (4.7 TB/s) with lengths from half to all, the fullest SM then having 1.5 times the
// mean.
//
// k_weights_many: a block keeps 128 keys in TMEM, as the first operand, and streams
// Q tiles (out of L2) past them, half a tile's scores (64 columns) in each of three
// buffers, so that the products run ahead of the exponentials.  Two blocks of eight
// exponential warps an SM: the unit takes 16 a cycle and SM, 448 cycles a half tile
// with one pair in eight on the multiply-add pipe, but a warp's loads, waits and
// sums around 32 exponentials a thread take as long, and only other warps fill
// them.  1024 rows of 32 heads over 16384 keys of 8: 190 us, 0.70 PFLOP/s (the
// unit alone 117).  It was 185 before double waits ordered the warp's memory (188) and
// rows of lse -inf were passed over (190); then, with 64 columns a warp and half as
// many warps, 214, with 256 keys a block and two groups of four warps 228.
//
// One warp copies, one issues the products.  Every wait is bounded; a block whose
// wait gives up waits for the copies and products that it has in flight (bounded as
// well) and ends, and dc_sync reports it.
#include <algorithm>

#include "dc_cache.cuh"
#include "dc_ring.h"
#include "dc_umma.cuh"

namespace {

using namespace dcc;
using dcu::F2;

constexpr int KEYS = 128;   // keys of a tile: the MMA's M
constexpr int COLS = 128;   // query rows of a tile: its N
constexpr int FEW_THREADS = 192;
constexpr int MANY_EVERY = 8;
constexpr int PANEL_BYTES = 128 * 128;
constexpr float LOG2E = 1.4426950408889634f;

constexpr int STAGES = 5;  // two blocks an SM hold at most 113 KB each
constexpr int FEW_BARS = 2 * STAGES + 6;
template <int NP>
constexpr int FEW_SMEM = (NP + STAGES) * PANEL_BYTES + COLS * 4 + COLS / 8 + FEW_BARS * 8 + 8;  // (and a slot for the TMEM address)

struct CwArgs {
  const void* k;
  const int32_t* lens;
  const float* lse;
  float* acc;
  int64_t k_seq, k_tok, k_head, acc_seq, acc_head;
  float c, decay;
  int rows, heads, kv_heads, group, hd, cache, causal;
  int tile_rows, tile_cols, col_tiles;  // rows and columns (rows x group) of a Q tile
  int chunk, splits;                    // keys of a block, blocks of a head
  int cols_mma;                         // the products' N
  int* status;
};

// Of 32 columns from c0, a bit for each that is not summed: before `from` (they do not
// see the key), from `cols` on, and those in `gaps`.
__device__ __forceinline__ uint32_t left_out(int c0, int from, int cols, uint32_t gaps) {
  if (from > c0) gaps |= from - c0 >= 32 ? ~0u : (1u << (from - c0)) - 1;
  if (cols < c0 + 32) gaps |= cols <= c0 ? ~0u : ~0u << (cols - c0);
  return gaps;
}
// The exponentials of columns c0.. + 31 of a tile (scores x, scales L) added to `part`,
// but for those left out: their scores may be anything, and NaN - inf is not -inf.
// `late`: a lane of the warp has a `from` above 0.  Every `EVERY`-th pair is taken on
// the multiply-add pipe.
template <int EVERY>
__device__ __forceinline__ void add_columns(F2 (&part)[4], const uint32_t (&x)[32], const float* L, float c, int c0,
                                            int from, int cols, bool late, uint32_t gaps) {
  if (late || gaps || c0 + 32 > cols) {
    const uint32_t out = left_out(c0, from, cols, gaps);
#pragma unroll
    for (int j = 0; j < 32; j++) {
      const float e = dcu::ex2(fmaf(__uint_as_float(x[j]), c, L[c0 + j]));
      part[j & 3] = dcu::add2(part[j & 3], dcu::f2(out & (1u << j) ? 0.0f : e, 0.0f));
    }
    return;
  }
  const F2 c2 = dcu::f2(c, c);
  const float4* l4 = reinterpret_cast<const float4*>(L + c0);
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float4 l = l4[j];
    const F2 lp[2] = {dcu::f2(l.x, l.y), dcu::f2(l.z, l.w)};
#pragma unroll
    for (int y = 0; y < 2; y++) {
      const int k = 4 * j + 2 * y;
      F2 e = dcu::fma2(dcu::f2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), c2, lp[y]);
      if ((2 * j + y) % EVERY == EVERY - 1) {
        e = dcu::ex2_fma(e);
      } else {
        const float2 v = dcu::split(e);
        e = dcu::f2(dcu::ex2(v.x), dcu::ex2(v.y));
      }
      part[(2 * j + y) & 3] = dcu::add2(part[(2 * j + y) & 3], e);
    }
  }
}
__device__ __forceinline__ float sum_of(const F2 (&part)[4]) {
  const float2 v = dcu::split(dcu::add2(dcu::add2(part[0], part[1]), dcu::add2(part[2], part[3])));
  return v.x + v.y;
}
// lse of column col of Q tile t (+inf: no row), and what is added to a column's
// exponents: -lse * log2 e, -inf where nothing is to be summed.
__device__ __forceinline__ float lse_of(const CwArgs& a, int64_t lse_at, int t, int col) {
  const int row = t * a.tile_rows + col / a.group;
  return col < a.tile_cols && row < a.rows ? a.lse[lse_at + (int64_t)row * a.heads + col % a.group] : INFINITY;
}
__device__ __forceinline__ float scale_of(float lse) { return lse == -INFINITY ? -INFINITY : -lse * LOG2E; }
__device__ __forceinline__ void put(const CwArgs& a, int b, int h, int key, float sum) {
  float* at = a.acc + b * a.acc_seq + h * a.acc_head + key;
  *at = a.decay == 0.0f ? sum : fmaf(a.decay, *at, sum);
}
// Panel rows that no Q copy writes (128 is no multiple of the group): zero, so
// that their scores are 0 and not what the memory held.
__device__ __forceinline__ void zero_rows(uint8_t* panels, int count, int tile_cols, int threads) {
  if (tile_cols >= COLS) return;
  const int per = (COLS - tile_cols) * 8;
  for (int i = threadIdx.x; i < per * count; i += threads) {
    const int p = i / per, rest = i - p * per;
    *reinterpret_cast<uint4*>(panels + p * PANEL_BYTES + tile_cols * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

template <int NP, bool BF16>
__global__ void __launch_bounds__(FEW_THREADS, 2)
    k_weights_few(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q,
                  const __grid_constant__ CwArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* kept = smem;
  uint8_t* ring = smem + NP * PANEL_BYTES;
  float* L = (float*)(ring + STAGES * PANEL_BYTES);  // the columns' scales
  uint32_t* gaps = (uint32_t*)(L + COLS);            // a bit for each column of lse -inf
  uint64_t* full = (uint64_t*)(gaps + COLS / 32);
  uint64_t* empty = full + STAGES;
  uint64_t* s_full = empty + STAGES;  // [2] scores of a buffer are in TMEM
  uint64_t* s_free = s_full + 2;      // [2] and have been read
  uint64_t* kept_full = s_free + 2;
  uint64_t* idle = kept_full + 1;  // all products that were issued are complete
  uint32_t* slot = (uint32_t*)(full + FEW_BARS);

  const int warp = dcu::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int split = blockIdx.x % a.splits, bg = blockIdx.x / a.splits;
  const int h = bg % a.kv_heads, b = bg / a.kv_heads;
  const int len = max(0, min(a.lens[b], a.cache));
  const int k0 = split * a.chunk, k1 = min(len, k0 + a.chunk);
  if (k1 <= k0) return;
  const int n = (k1 - k0 + KEYS - 1) / KEYS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; i++) {
      dcp::mbar_init(&full[i], 1);
      dcp::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      dcp::mbar_init(&s_full[i], 1);
      dcp::mbar_init(&s_free[i], 4);
    }
    dcp::mbar_init(kept_full, 1);
    dcp::mbar_init(idle, 1);
    dcp::mbar_fence_init();
  }
  if (warp == 5) dcu::alloc(slot, 2 * COLS);
  zero_rows(kept, NP, a.tile_cols, FEW_THREADS);
  float lse = INFINITY;
  if (threadIdx.x < COLS) {
    lse = lse_of(a, (int64_t)b * a.rows * a.heads + h * a.group, 0, threadIdx.x);
    L[threadIdx.x] = scale_of(lse);
  }
  dcu::fence_before();
  const uint32_t gap = __ballot_sync(~0u, lse == -INFINITY);
  if (threadIdx.x < COLS && lane == 0) gaps[warp] = gap;
  __syncthreads();
  dcu::fence_after();
  const uint32_t tmem = dcu::uniform(*slot);
  // (only now: a dependent that takes TMEM before its own wait must not take
  // what a block of this grid still has to get)
  asm volatile("griddepcontrol.launch_dependents;");

  if (warp == 4) {
    if (lane == 0) {
      dcp::mbar_expect_tx(kept_full, NP * a.tile_cols * 128);
#pragma unroll
      for (int p = 0; p < NP; p++) dcu::tma_load_5d(kept + p * PANEL_BYTES, &map_q, p * 64, 0, h, 0, b, kept_full);
      int issued = 0;
      for (int s = 0; s < n * NP; s++, issued++) {
        const int st = s % STAGES, i = s / NP, p = s - i * NP;
        if (s >= STAGES && !dcp::mbar_wait(&empty[st], ((s / STAGES) & 1) ^ 1, a.status)) break;
        dcp::mbar_expect_tx(&full[st], PANEL_BYTES);
        dcu::tma_load_4d(ring + st * PANEL_BYTES, &map_k, p * 64, h, k0 + i * KEYS, b, &full[st]);
      }
      dcp::mbar_wait(kept_full, 0, a.status);
      dcr::drain<STAGES>(issued, [&](int st, uint32_t par) { dcp::mbar_wait(&full[st], par, a.status); });
    }
  } else if (warp == 5) {
    const uint32_t id = dcu::idesc(BF16, 0, false) | ((uint32_t)(a.cols_mma >> 3) << 17);
    const uint64_t dq = dcu::desc(dcp::smem_u32(kept), 0), dk = dcu::desc(dcp::smem_u32(ring), 0);
    bool ok = dcu::warp_wait(kept_full, 0, a.status);
    for (int i = 0; i < n && ok; i++) {
      if (i >= 2) ok = dcu::warp_wait(&s_free[i & 1], ((i >> 1) & 1) ^ 1, a.status);
#pragma unroll
      for (int p = 0; p < NP; p++) {
        const int s = i * NP + p, st = s % STAGES;
        ok = ok && dcu::warp_wait(&full[st], (s / STAGES) & 1, a.status);
        if (!ok) break;
        dcu::fence_after();
        if (dcu::elect()) {
#pragma unroll
          for (int kk = 0; kk < 4; kk++)
            dcu::mma_ss(tmem + (i & 1) * COLS, dk + st * (PANEL_BYTES >> 4) + kk * 2, dq + p * (PANEL_BYTES >> 4) + kk * 2,
                        id, p > 0 || kk > 0);
          dcu::commit(&empty[st]);
          if (p == NP - 1) dcu::commit(&s_full[i & 1]);
        }
        __syncwarp();
      }
    }
    // (also where a wait gave up: nothing reads shared memory or writes TMEM any more)
    if (dcu::elect()) dcu::commit(idle);
    __syncwarp();
    dcu::warp_wait(idle, 0, a.status);
  } else {
    const uint32_t lane_at = tmem + ((uint32_t)(warp * 32) << 16);
    const int cols = a.tile_cols;
    for (int i = 0; i < n; i++) {
      if (!dcu::warp_wait(&s_full[i & 1], (i >> 1) & 1, a.status)) break;
      dcu::fence_after();
      const int key = k0 + i * KEYS + warp * 32 + lane;
      const int from = a.causal ? max(0, key - len + a.rows) * a.group : 0;  // columns that see the key
      const bool late = __any_sync(~0u, from > 0);
      F2 part[4] = {dcu::f2(0, 0), dcu::f2(0, 0), dcu::f2(0, 0), dcu::f2(0, 0)};
#pragma unroll 1
      for (int c0 = 0; c0 < cols; c0 += 32) {
        uint32_t x[32];
        const uint32_t gap = gaps[c0 / 32];
        dcu::ld32(lane_at + (i & 1) * COLS + c0, x);
        dcu::wait_ld(x);
        add_columns<1 << 20>(part, x, L, a.c, c0, from, cols, late, gap);
      }
      dcu::fence_before();
      __syncwarp();
      if (lane == 0) dcp::mbar_arrive(&s_free[i & 1]);
      if (key < k1) put(a, b, h, key, sum_of(part));
    }
  }
  __syncthreads();
  if (warp == 5) {
    dcu::fence_after();
    dcu::dealloc(tmem, 2 * COLS);
  }
}

// Blocks of 128 keys against all Q tiles, two an SM, a half tile (64 columns) at a
// time.  TMEM columns: the keys (64 x 32 bits a lane), three half tiles' scores.
// (One pair in eight by multiply-adds: 185 us, then; in six 186, in twelve 192, in
// four 200, none 196.)
constexpr int HALF = COLS / 2, BUFS = 3, SCALES = 4;
constexpr int MANY_THREADS = 352, MMA_WARP = 0, TMA_WARP = 1, SCALE_WARP = 2, EXP_WARP = 3;
constexpr uint32_t s_col(int i) { return 64 + i * HALF; }
template <int NP>
struct Many {
  static constexpr int TILE = NP * PANEL_BYTES;
  static constexpr int STAGES = NP == 2 ? 3 : 6;
  static constexpr int BARS = 2 * STAGES + 2 * BUFS + 2 * SCALES + 2;
  static constexpr int SMEM = STAGES * TILE + SCALES * COLS * 4 + KEYS * 4 + SCALES * COLS / 8 + BARS * 8 + 8;
};

template <int NP, bool BF16>
__global__ void __launch_bounds__(MANY_THREADS, 2)
    k_weights_many(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CwArgs a) {
  using C = Many<NP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem;
  float* scales = (float*)(ring + C::STAGES * C::TILE);  // [SCALES tiles][COLS]
  float* halves = scales + SCALES * COLS;                // [KEYS] sums of the second warps
  uint32_t* gaps = (uint32_t*)(halves + KEYS);           // [SCALES tiles] a bit for each column of lse -inf
  uint64_t* full = (uint64_t*)(gaps + SCALES * COLS / 32);
  uint64_t* empty = full + C::STAGES;
  uint64_t* s_full = empty + C::STAGES;  // [BUFS] a half tile's scores are in TMEM
  uint64_t* s_free = s_full + BUFS;      // [BUFS] and have been read
  uint64_t* l_full = s_free + BUFS;      // [SCALES] a tile's scales are there
  uint64_t* l_free = l_full + SCALES;    // [SCALES] and have been read
  uint64_t* k_ready = l_free + SCALES;   // the keys are in TMEM
  uint64_t* idle = k_ready + 1;          // all products that were issued are complete
  uint32_t* slot = (uint32_t*)(full + C::BARS);

  const int warp = dcu::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int split = blockIdx.x % a.splits, bg = blockIdx.x / a.splits;
  const int h = bg % a.kv_heads, b = bg / a.kv_heads;
  const int len = max(0, min(a.lens[b], a.cache));
  const int k0 = split * KEYS;
  if (len <= k0) return;
  // Q tiles from the first that holds a row which sees the block's first key
  const int t0 = a.causal ? max(0, k0 - len + a.rows) / a.tile_rows : 0, n = a.col_tiles - t0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; i++) {
      dcp::mbar_init(&full[i], 1);
      dcp::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < BUFS; i++) {
      dcp::mbar_init(&s_full[i], 1);
      dcp::mbar_init(&s_free[i], 8);
    }
    for (int i = 0; i < SCALES; i++) {
      dcp::mbar_init(&l_full[i], 1);
      dcp::mbar_init(&l_free[i], 8);
    }
    dcp::mbar_init(k_ready, 8);
    dcp::mbar_init(idle, 1);
    dcp::mbar_fence_init();
  }
  if (warp == MMA_WARP) dcu::alloc(slot, 256);
  zero_rows(ring, C::STAGES * NP, a.tile_cols, MANY_THREADS);
  dcu::fence_before();
  __syncthreads();
  dcu::fence_after();
  const uint32_t tmem = dcu::uniform(*slot);
  // (only now: see k_weights_few)
  asm volatile("griddepcontrol.launch_dependents;");

  if (warp == TMA_WARP) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < n; i++, issued++) {
        const int st = i % C::STAGES;
        if (i >= C::STAGES && !dcp::mbar_wait(&empty[st], ((i / C::STAGES) & 1) ^ 1, a.status)) break;
        dcp::mbar_expect_tx(&full[st], NP * a.tile_cols * 128);
#pragma unroll
        for (int p = 0; p < NP; p++)
          dcu::tma_load_5d(ring + st * C::TILE + p * PANEL_BYTES, &map_q, p * 64, 0, h, (t0 + i) * a.tile_rows, b, &full[st]);
      }
      dcr::drain<C::STAGES>(issued, [&](int st, uint32_t par) { dcp::mbar_wait(&full[st], par, a.status); });
    }
  } else if (warp == MMA_WARP) {
    const uint32_t id = dcu::idesc(BF16, HALF, false);
    const uint64_t dq = dcu::desc(dcp::smem_u32(ring), 0);
    bool ok = dcu::warp_wait(k_ready, 0, a.status);
    for (int u = 0; u < 2 * n && ok; u++) {
      const int i = u >> 1, st = i % C::STAGES, buf = u % BUFS;
      // (lanes by turns: the tile is here, the scores before have been read)
      const bool odd = (lane & 1) && u >= BUFS;
      ok = dcu::warp_wait_each(odd ? &s_free[buf] : &full[st], odd ? (u / BUFS - 1) & 1 : (i / C::STAGES) & 1, a.status);
      if (!ok) break;
      dcu::fence_after();
      if (dcu::elect()) {
#pragma unroll
        for (int kk = 0; kk < 4 * NP; kk++)
          dcu::mma_ts(tmem + s_col(buf), tmem + kk * 8,
                      dq + ((st * C::TILE + (u & 1) * HALF * 128 + (kk >> 2) * PANEL_BYTES + (kk & 3) * 32) >> 4), id, kk > 0);
        dcu::commit(&s_full[buf]);
        if (u & 1) dcu::commit(&empty[st]);
      }
      __syncwarp();
    }
    // (also where a wait gave up: nothing reads shared memory or writes TMEM any more)
    if (dcu::elect()) dcu::commit(idle);
    __syncwarp();
    dcu::warp_wait(idle, 0, a.status);
  } else if (warp == SCALE_WARP) {
    // ---- each Q tile's scales, a tile's lse read while the one before is waited for
    const int64_t lse_at = (int64_t)b * a.rows * a.heads + h * a.group;
    float next[COLS / 32];
#pragma unroll
    for (int x = 0; x < COLS / 32; x++) next[x] = lse_of(a, lse_at, t0, x * 32 + lane);
    for (int i = 0; i < n; i++) {
      const int st = i % SCALES;
      if (i >= SCALES && !dcu::warp_wait(&l_free[st], ((i / SCALES) & 1) ^ 1, a.status)) break;
#pragma unroll
      for (int x = 0; x < COLS / 32; x++) {
        scales[st * COLS + x * 32 + lane] = scale_of(next[x]);
        const uint32_t gap = __ballot_sync(~0u, next[x] == -INFINITY);
        if (lane == 0) gaps[st * (COLS / 32) + x] = gap;
        if (i + 1 < n) next[x] = lse_of(a, lse_at, t0 + i + 1, x * 32 + lane);
      }
      __syncwarp();
      if (lane == 0) dcp::mbar_arrive(&l_full[st]);
    }
  } else {
    const int quarter = warp & 3, half = (warp - EXP_WARP) >> 2;  // TMEM lanes, half of a buffer's columns
    const uint32_t lane_at = tmem + ((uint32_t)(quarter * 32) << 16);
    const int key = k0 + quarter * 32 + lane;
    // ---- this thread's key into TMEM (once a block; zeros behind the cache's end)
    {
      const uint4* src = (const uint4*)((const uint16_t*)a.k + b * a.k_seq + (int64_t)key * a.k_tok + h * a.k_head);
#pragma unroll
      for (int p = 0; p < NP; p++) {
        if (p != half) continue;
        uint32_t r[32];
#pragma unroll
        for (int x = 0; x < 8; x++) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (key < a.cache && (8 * p + x) * 8 < a.hd) v = src[8 * p + x];
          r[4 * x] = v.x, r[4 * x + 1] = v.y, r[4 * x + 2] = v.z, r[4 * x + 3] = v.w;
        }
        dcu::st32(lane_at + 32 * p, r);
      }
      dcu::wait_st();
      dcu::fence_before();
      __syncwarp();
      if (lane == 0) dcp::mbar_arrive(k_ready);
    }
    const int hidden = a.causal ? key - len + a.rows : 0;  // rows that do not see the key
    float sum = 0.0f;
    bool ok = true;
#pragma unroll 1
    for (int u = 0; u < 2 * n; u++) {
      const int i = u >> 1, st = i % SCALES, buf = u % BUFS;
      const bool odd = lane & 1;
      ok = dcu::warp_wait_each(odd ? &l_full[st] : &s_full[buf], odd ? (i / SCALES) & 1 : (u / BUFS) & 1, a.status);
      if (!ok) break;
      dcu::fence_after();
      const int first_row = (t0 + i) * a.tile_rows, c0 = (u & 1) * HALF + half * 32;
      const int cols = min(a.tile_cols, (a.rows - first_row) * a.group);
      const bool late = __any_sync(~0u, hidden > first_row);
      const int from = late ? max(0, hidden - first_row) * a.group : 0;  // columns that see the key
      F2 part[4] = {dcu::f2(0, 0), dcu::f2(0, 0), dcu::f2(0, 0), dcu::f2(0, 0)};
      const float* L = scales + st * COLS;
      const uint32_t gap = gaps[st * (COLS / 32) + c0 / 32];
      uint32_t x[32];
      dcu::ld32(lane_at + s_col(buf) + half * 32, x);
      dcu::wait_ld(x);
      dcu::fence_before();
      __syncwarp();
      if (lane == 0) dcp::mbar_arrive(&s_free[buf]);
      if (c0 < cols) add_columns<MANY_EVERY>(part, x, L, a.c, c0, from, cols, late, gap);
      sum += sum_of(part);
      __syncwarp();
      if ((u & 1) && lane == 0) dcp::mbar_arrive(&l_free[st]);
    }
    if (half) halves[quarter * 32 + lane] = ok ? sum : -1.0f;
    dcp::named_sync(1, 256);
    const float other = halves[quarter * 32 + lane];
    if (!half && ok && key < len && other != -1.0f) put(a, b, h, key, sum + other);
  }
  __syncthreads();
  if (warp == MMA_WARP) {
    dcu::fence_after();
    dcu::dealloc(tmem, 256);
  }
}

template <int NP, bool BF16>
int run(dc_ctx* ctx, const CUtensorMap& k, const CUtensorMap& q, const CwArgs& a, int64_t blocks, bool few) {
  const dim3 grid((unsigned)blocks);
  return few ? launch(ctx, k_weights_few<NP, BF16>, grid, FEW_THREADS, FEW_SMEM<NP>, 1, k, q, a)
             : launch(ctx, k_weights_many<NP, BF16>, grid, MANY_THREADS, Many<NP>::SMEM, 1, q, a);
}

}  // namespace

extern "C" int dc_cache_weights_dev(dc_ctx* ctx, const dc_cache_weight* p) {
  if (!ctx || !p) return dc_fail(ctx, DC_E_INVAL, "cache_weights: bad arguments");
  const dc_cache_weight& A = *p;
  if (A.batch < 0 || A.rows < 1 || A.heads < 1 || A.kv_heads < 1 || A.heads % A.kv_heads ||
      A.heads / A.kv_heads > COLS)
    return dc_fail(ctx, DC_E_INVAL, "cache_weights: batch %d, rows %d, heads %d of %d (at most %d a head)", A.batch,
                   A.rows, A.heads, A.kv_heads, COLS);
  if (A.head_dim < 8 || A.head_dim > 128 || (A.head_dim & 7))
    return dc_fail(ctx, DC_E_INVAL, "cache_weights: head_dim %d must be a multiple of 8 up to 128", A.head_dim);
  if (A.cache < 0 || A.cache > (1 << 30) || A.rows > (1 << 22) || (int64_t)A.batch * A.kv_heads > (1 << 20))
    return dc_fail(ctx, DC_E_INVAL, "cache_weights: cache %d, rows %d, batch %d", A.cache, A.rows, A.batch);
  if (!is_half(A.type)) return dc_fail(ctx, DC_E_INVAL, "cache_weights: type f16 or bf16");
  const float c = (float)(A.scale * 1.4426950408889634);
  if (!(c > 0.0f) || !isfinite(c)) return dc_fail(ctx, DC_E_INVAL, "cache_weights: scale %g", A.scale);
  if (!isfinite((float)A.decay)) return dc_fail(ctx, DC_E_INVAL, "cache_weights: decay %g", A.decay);
  if (!A.batch || !A.cache) return DC_OK;
  if (!A.q || !A.k || !A.lens || !A.lse || !A.acc) return dc_fail(ctx, DC_E_INVAL, "cache_weights: null buffer");
  if (!aligned(A.q, 2, 16, {{A.batch, A.q_seq}, {A.rows, A.q_row}, {A.heads, A.q_head}}) ||
      !aligned(A.k, 2, 16, {{A.batch, A.k_seq}, {A.cache, A.k_tok}, {A.kv_heads, A.k_head}}))
    return dc_fail(ctx, DC_E_INVAL, "cache_weights: q and k rows must begin on 16-byte boundaries");
  const std::initializer_list<Dim> d_acc = {{A.batch, A.acc_seq}, {A.kv_heads, A.acc_head}, {A.cache, 1}};
  const Span acc = span(A.acc, 4, d_acc);
  const Span in[4] = {span(A.q, 2, {{A.batch, A.q_seq}, {A.rows, A.q_row}, {A.heads, A.q_head}, {A.head_dim, 1}}),
                      span(A.k, 2, {{A.batch, A.k_seq}, {A.cache, A.k_tok}, {A.kv_heads, A.k_head}, {A.head_dim, 1}}),
                      span(A.lse, 4, {{(int64_t)A.batch * A.rows * A.heads, 1}}), span(A.lens, 4, {{A.batch, 1}})};
  for (const Span& s : in)
    if (!acc.ok || !s.ok || acc.meets(s))
      return dc_fail(ctx, DC_E_INVAL, "cache_weights: a negative stride, or acc overlaps an input");
  if (!apart(d_acc)) return dc_fail(ctx, DC_E_INVAL, "cache_weights: two elements of acc share an address");
  DeviceGuard guard;
  if (int rc = guard.enter(ctx)) return rc;

  CwArgs a;
  a.group = A.heads / A.kv_heads;
  a.tile_rows = COLS / a.group;
  const bool few = A.rows <= a.tile_rows;
  if (few) a.tile_rows = A.rows;
  a.tile_cols = a.tile_rows * a.group;
  a.col_tiles = (A.rows + a.tile_rows - 1) / a.tile_rows;
  a.cols_mma = (a.tile_cols + 31) / 32 * 32;  // (columns are read 32 at a time)
  const int64_t heads = (int64_t)A.batch * A.kv_heads, tiles = (A.cache + KEYS - 1) / KEYS;
  // few: one wave of two blocks an SM, each an even share of a head's key
  // tiles; many: a block for every key tile
  int64_t splits = tiles;
  if (few) {
    splits = std::min(tiles, std::max<int64_t>(1, 2 * (int64_t)ctx->sm_count / heads));
    const int64_t each = (tiles + splits - 1) / splits;
    splits = (tiles + each - 1) / each;
    a.chunk = (int)(each * KEYS);
  }
  a.splits = (int)splits;
  if (heads * splits > INT32_MAX) return dc_fail(ctx, DC_E_INVAL, "cache_weights: too many blocks");

  const bool bf16 = A.type == DC_BF16;
  CUtensorMap mk, mq;
  const uint64_t dk[4] = {(uint64_t)A.head_dim, (uint64_t)A.kv_heads, (uint64_t)A.cache, (uint64_t)A.batch};
  const uint64_t sk[3] = {2 * (uint64_t)A.k_head, 2 * (uint64_t)A.k_tok, 2 * (uint64_t)A.k_seq};
  const uint32_t bk[4] = {64, 1, KEYS, 1};
  const uint64_t dq[5] = {(uint64_t)A.head_dim, (uint64_t)a.group, (uint64_t)A.kv_heads, (uint64_t)A.rows,
                          (uint64_t)A.batch};
  const uint64_t sq[4] = {2 * (uint64_t)A.q_head, 2 * (uint64_t)A.q_head * a.group, 2 * (uint64_t)A.q_row,
                          2 * (uint64_t)A.q_seq};
  const uint32_t bq[5] = {64, (uint32_t)a.group, 1, (uint32_t)a.tile_rows, 1};
  if (!dcu::encode(&mk, A.k, bf16, 4, dk, sk, bk) || !dcu::encode(&mq, A.q, bf16, 5, dq, sq, bq))
    return dc_fail(ctx, DC_E_INVAL, "cache_weights: these q or k strides make no tensor map");
  a.k = A.k, a.k_seq = A.k_seq, a.k_tok = A.k_tok, a.k_head = A.k_head, a.hd = A.head_dim;
  a.lens = A.lens, a.lse = A.lse, a.acc = A.acc, a.acc_seq = A.acc_seq, a.acc_head = A.acc_head;
  a.c = c, a.decay = (float)A.decay;
  a.rows = A.rows, a.heads = A.heads, a.kv_heads = A.kv_heads, a.cache = A.cache, a.causal = A.causal != 0;
  a.status = ctx->d_status;
  if (A.head_dim <= 64)
    return bf16 ? run<1, true>(ctx, mk, mq, a, heads * splits, few)
                : run<1, false>(ctx, mk, mq, a, heads * splits, few);
  return bf16 ? run<2, true>(ctx, mk, mq, a, heads * splits, few)
              : run<2, false>(ctx, mk, mq, a, heads * splits, few);
}
