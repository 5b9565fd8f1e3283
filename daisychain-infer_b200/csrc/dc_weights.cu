// dc_weights.cu -- the softmax weight that every cached key receives.
//
//   acc[b][g][j] = decay acc[b][g][j] + sum over rows r and heads h of group g of exp(scale q_rh . k_j - lse_rh)
//
// With lse known the sum needs no running maximum and no second pass.  The
// product is formed as K Q^T: keys on the 128 TMEM lanes, up to 128 query rows
// (row, head of the group; heads innermost) on the columns.  A thread then holds
// one key against all rows and adds its exponentials in a register: no
// exchange, no atomics, one order of summation.
//
// Few rows (one column tile): a block keeps Q and streams its share of the
// cache's keys; HBM-bound, each key is read once.  Many rows: a block keeps 128
// keys and streams Q tiles (out of L2) past them; bound by the exponential unit,
// 16 a cycle and SM: 128 x 128 of them take 1024 cycles, their products 512.
// Two blocks share an SM, and the scores are double-buffered in TMEM, so copies
// and products run under the exponentials.
//
// Warps 0-3 own a TMEM lane (key) per thread, warp 4 copies 64-element panels
// (16 KB) into a ring by TMA, warp 5 issues the products.  Every wait is
// bounded; a block whose wait gives up ends, and dc_sync reports it.
#include <algorithm>

#include "dc_cache.cuh"
#include "dc_umma.cuh"

namespace {

using namespace dcc;
using dcu::F2;

constexpr int KEYS = 128;   // keys of a tile: the MMA's M
constexpr int COLS = 128;   // query rows of a tile: its N
constexpr int THREADS = 192;
constexpr int PANEL_BYTES = 128 * 128;
constexpr uint32_t TMEM_COLS = 256;  // two buffers of COLS scores
constexpr float LOG2E = 1.4426950408889634f;

// Two blocks an SM hold at most 113 KB each: beside two panels of the kept tile
// and the scales, five ring stages or (two buffers of scales) four.
template <int NP, bool KEEP_Q>
struct Cfg {
  static constexpr int STAGES = KEEP_Q || NP == 1 ? 5 : 4;
  static constexpr int SCALES = KEEP_Q ? 1 : 2;
  static constexpr int SMEM = (NP + STAGES) * PANEL_BYTES + SCALES * COLS * 4 + 128;
};

struct CwArgs {
  const int32_t* lens;
  const float* lse;
  float* acc;
  int64_t acc_seq, acc_head;
  float c, decay;
  int rows, heads, kv_heads, group, cache, causal;
  int tile_rows, tile_cols, col_tiles;  // rows and columns (rows x group) of a Q tile
  int chunk, splits;                    // keys of a block, blocks of a head
  int cols_mma;                         // the products' N
  int* status;
};

// KEEP_Q: the block keeps its one Q tile and streams keys; otherwise it keeps
// its one key tile and streams Q tiles.
template <int NP, bool BF16, bool KEEP_Q>
__global__ void __launch_bounds__(THREADS, 2)
    k_cache_weights(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q,
                    const __grid_constant__ CwArgs a) {
  using C = Cfg<NP, KEEP_Q>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* kept = smem;
  uint8_t* ring = smem + NP * PANEL_BYTES;
  float* scales = (float*)(ring + STAGES * PANEL_BYTES);  // -lse * log2 e of a tile's columns; -inf where nothing is added
  uint64_t* full = (uint64_t*)(scales + C::SCALES * COLS);
  uint64_t* empty = full + STAGES;
  uint64_t* s_full = empty + STAGES;  // [2] scores of a buffer are in TMEM
  uint64_t* s_free = s_full + 2;      // [2] and have been read
  uint64_t* kept_full = s_free + 2;
  uint32_t* slot = (uint32_t*)(kept_full + 1);

  const int warp = dcu::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int split = blockIdx.x % a.splits, bg = blockIdx.x / a.splits;
  const int h = bg % a.kv_heads, b = bg / a.kv_heads;
  const int len = max(0, min(a.lens[b], a.cache));
  const int k0 = split * a.chunk, k1 = min(len, k0 + a.chunk);
  if (k1 <= k0) return;
  // (key tile, Q tile) pairs in turn: KEEP_Q walks the keys, else the Q tiles,
  // from the first that holds a row which sees the block's first key
  const int see0 = a.causal ? max(0, k0 - len + a.rows) : 0;  // first row that sees key k0
  const int t0 = KEEP_Q ? 0 : see0 / a.tile_rows;
  const int n = KEEP_Q ? (k1 - k0 + KEYS - 1) / KEYS : a.col_tiles - t0;

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
    dcp::mbar_fence_init();
  }
  if (warp == 5) dcu::alloc(slot, TMEM_COLS);
  // panel rows that no Q copy writes (128 is no multiple of the group): zero,
  // so that their scores are 0 and not what the memory held
  if (a.tile_cols < COLS) {
    uint8_t* at = KEEP_Q ? kept : ring;
    const int per = (COLS - a.tile_cols) * 8, panels = KEEP_Q ? NP : STAGES;
    for (int i = threadIdx.x; i < per * panels; i += THREADS) {
      const int p = i / per, rest = i - p * per;
      *reinterpret_cast<uint4*>(at + p * PANEL_BYTES + a.tile_cols * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  dcu::fence_before();
  __syncthreads();
  dcu::fence_after();
  const uint32_t tmem = dcu::uniform(*slot);
  // (only now: a dependent that takes TMEM before its own wait must not take
  // what a block of this grid still has to get)
  asm volatile("griddepcontrol.launch_dependents;");

  const int q_bytes = a.tile_cols * 128;
  if (warp == 4) {
    if (lane == 0) {
      const int kept_bytes = KEEP_Q ? q_bytes : PANEL_BYTES, ring_bytes = KEEP_Q ? PANEL_BYTES : q_bytes;
      dcp::mbar_expect_tx(kept_full, NP * kept_bytes);
#pragma unroll
      for (int p = 0; p < NP; p++) {
        if (KEEP_Q)
          dcu::tma_load_5d(kept + p * PANEL_BYTES, &map_q, p * 64, 0, h, 0, b, kept_full);
        else
          dcu::tma_load_4d(kept + p * PANEL_BYTES, &map_k, p * 64, h, k0, b, kept_full);
      }
      int issued = 0;
      for (int s = 0; s < n * NP; s++, issued++) {
        const int st = s % STAGES, i = s / NP, p = s - i * NP;
        if (s >= STAGES && !dcp::mbar_wait(&empty[st], ((s / STAGES) & 1) ^ 1, a.status)) break;
        dcp::mbar_expect_tx(&full[st], ring_bytes);
        uint8_t* dst = ring + st * PANEL_BYTES;
        if (KEEP_Q)
          dcu::tma_load_4d(dst, &map_k, p * 64, h, k0 + i * KEYS, b, &full[st]);
        else
          dcu::tma_load_5d(dst, &map_q, p * 64, 0, h, (t0 + i) * a.tile_rows, b, &full[st]);
      }
      if (issued < n * NP) {
        // (given up: what is in flight lands before the block's memory goes away)
        dcp::mbar_wait(kept_full, 0, a.status);
        for (int s = max(0, issued - STAGES); s < issued; s++)
          dcp::mbar_wait(&full[s % STAGES], (s / STAGES) & 1, a.status);
      }
    }
  } else if (warp == 5) {
    {
      const uint32_t id = dcu::idesc(BF16, 0, false) | ((uint32_t)(a.cols_mma >> 3) << 17);
      const uint32_t kept_at = dcp::smem_u32(kept), ring_at = dcp::smem_u32(ring);
      bool ok = __all_sync(~0u, dcp::mbar_wait(kept_full, 0, a.status));
      for (int i = 0; i < n && ok; i++) {
        if (i >= 2) ok = __all_sync(~0u, dcp::mbar_wait(&s_free[i & 1], ((i >> 1) & 1) ^ 1, a.status));
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const int s = i * NP + p, st = s % STAGES;
          ok = ok && __all_sync(~0u, dcp::mbar_wait(&full[st], (s / STAGES) & 1, a.status));
          if (!ok) break;
          dcu::fence_after();
          const uint32_t keep = kept_at + p * PANEL_BYTES, move = ring_at + st * PANEL_BYTES;
          const uint64_t dkeep = dcu::desc(keep, 0), dmove = dcu::desc(move, 0);
          if (dcu::elect()) {
#pragma unroll
            for (int kk = 0; kk < 4; kk++)
              dcu::mma_ss(tmem + (i & 1) * COLS, (KEEP_Q ? dmove : dkeep) + kk * 2, (KEEP_Q ? dkeep : dmove) + kk * 2, id,
                          p > 0 || kk > 0);
            dcu::commit(&empty[st]);
            if (p == NP - 1) dcu::commit(&s_full[i & 1]);
          }
          __syncwarp();
        }
      }
    }
  } else {
    const uint32_t lane_at = tmem + ((uint32_t)(warp * 32) << 16);
    const int64_t lse_at = (int64_t)b * a.rows * a.heads + h * a.group;
    // column `threadIdx.x` of Q tile t
    auto column = [&](int t) {
      const int col = threadIdx.x, row = t * a.tile_rows + col / a.group;
      float v = -INFINITY;
      if (col < a.tile_cols && row < a.rows) {
        v = -a.lse[lse_at + (int64_t)row * a.heads + col % a.group] * LOG2E;
        if (v == INFINITY) v = -INFINITY;
      }
      return v;
    };
    float next = column(t0);
    float sum = 0.0f;
    bool ok = true;  // (a warp whose wait gave up stays in the loop: the others count on it at the barrier)
    for (int i = 0; i < n; i++) {
      float* L = scales + (KEEP_Q ? 0 : (i & 1) * COLS);
      if (!KEEP_Q || i == 0) {
        L[threadIdx.x] = next;
        if (!KEEP_Q && i + 1 < n) next = column(t0 + i + 1);
        // (one barrier a tile: who passes it has read the buffer of two tiles ago)
        dcp::named_sync(1, 128);
      }
      ok = ok && __all_sync(~0u, dcp::mbar_wait(&s_full[i & 1], (i >> 1) & 1, a.status));
      if (!ok) continue;
      dcu::fence_after();
      const int key = (KEEP_Q ? k0 + i * KEYS : k0) + warp * 32 + lane;
      const int first_row = KEEP_Q ? 0 : (t0 + i) * a.tile_rows;
      // columns of this tile that see the key
      const int from = a.causal ? max(0, (key - len + a.rows - first_row)) * a.group : 0;
      const int cols = min(a.tile_cols, (a.rows - first_row) * a.group);
      const bool late = __any_sync(~0u, from > 0);
      if (KEEP_Q) sum = 0.0f;
      const F2 c2 = dcu::f2(a.c, a.c);
      F2 part[4] = {dcu::f2(0, 0), dcu::f2(0, 0), dcu::f2(0, 0), dcu::f2(0, 0)};
      uint32_t s[2][32];
      // columns c0 .. c0 + 31, and the next ones' load meanwhile
      auto add = [&](uint32_t (&x)[32], uint32_t (&next)[32], int c0) {
        dcu::wait_ld(x);
        if (c0 + 32 < cols) dcu::ld32(lane_at + (i & 1) * COLS + c0 + 32, next);
        const float4* l4 = reinterpret_cast<const float4*>(L + c0);
        if (late || c0 + 32 > cols) {
#pragma unroll
          for (int j = 0; j < 32; j++) {
            const float e = dcu::ex2(fmaf(__uint_as_float(x[j]), a.c, L[c0 + j]));
            part[j & 3] = dcu::add2(part[j & 3], dcu::f2(c0 + j < from || c0 + j >= cols ? 0.0f : e, 0.0f));
          }
          return;
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float4 l = l4[j];
          const float2 t0 = dcu::split(
              dcu::fma2(dcu::f2(__uint_as_float(x[4 * j]), __uint_as_float(x[4 * j + 1])), c2, dcu::f2(l.x, l.y)));
          const float2 t1 = dcu::split(
              dcu::fma2(dcu::f2(__uint_as_float(x[4 * j + 2]), __uint_as_float(x[4 * j + 3])), c2, dcu::f2(l.z, l.w)));
          part[(2 * j) & 3] = dcu::add2(part[(2 * j) & 3], dcu::f2(dcu::ex2(t0.x), dcu::ex2(t0.y)));
          part[(2 * j + 1) & 3] = dcu::add2(part[(2 * j + 1) & 3], dcu::f2(dcu::ex2(t1.x), dcu::ex2(t1.y)));
        }
      };
      dcu::ld32(lane_at + (i & 1) * COLS, s[0]);
#pragma unroll 1
      for (int c0 = 0; c0 < cols; c0 += 64) {
        add(s[0], s[1], c0);
        if (c0 + 32 < cols) add(s[1], s[0], c0 + 32);
      }
      const float2 got = dcu::split(dcu::add2(dcu::add2(part[0], part[1]), dcu::add2(part[2], part[3])));
      sum += got.x + got.y;
      dcu::fence_before();
      __syncwarp();
      if (lane == 0) dcp::mbar_arrive(&s_free[i & 1]);
      if ((KEEP_Q || i == n - 1) && key < k1) {
        float* at = a.acc + b * a.acc_seq + h * a.acc_head + key;
        *at = a.decay == 0.0f ? sum : fmaf(a.decay, *at, sum);
      }
    }
  }
  __syncthreads();
  if (warp == 5) {
    dcu::fence_after();
    dcu::dealloc(tmem, TMEM_COLS);
  }
}

template <int NP, bool BF16>
int run(dc_ctx* ctx, const CUtensorMap& k, const CUtensorMap& q, const CwArgs& a, int64_t blocks, bool keep_q) {
  const dim3 grid((unsigned)blocks);
  return keep_q ? launch(ctx, k_cache_weights<NP, BF16, true>, grid, THREADS, Cfg<NP, true>::SMEM, 1, k, q, a)
                : launch(ctx, k_cache_weights<NP, BF16, false>, grid, THREADS, Cfg<NP, false>::SMEM, 1, k, q, a);
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
  const Span acc = span(A.acc, 4, {{A.batch, A.acc_seq}, {A.kv_heads, A.acc_head}, {A.cache, 1}});
  const Span in[4] = {span(A.q, 2, {{A.batch, A.q_seq}, {A.rows, A.q_row}, {A.heads, A.q_head}, {A.head_dim, 1}}),
                      span(A.k, 2, {{A.batch, A.k_seq}, {A.cache, A.k_tok}, {A.kv_heads, A.k_head}, {A.head_dim, 1}}),
                      span(A.lse, 4, {{(int64_t)A.batch * A.rows * A.heads, 1}}), span(A.lens, 4, {{A.batch, 1}})};
  for (const Span& s : in)
    if (!acc.ok || !s.ok || acc.meets(s))
      return dc_fail(ctx, DC_E_INVAL, "cache_weights: a negative stride, or acc overlaps an input");
  DeviceGuard guard;
  if (int rc = guard.enter(ctx)) return rc;

  CwArgs a;
  a.group = A.heads / A.kv_heads;
  a.tile_rows = COLS / a.group;
  const bool keep_q = A.rows <= a.tile_rows;
  if (keep_q) a.tile_rows = A.rows;
  a.tile_cols = a.tile_rows * a.group;
  a.col_tiles = (A.rows + a.tile_rows - 1) / a.tile_rows;
  a.cols_mma = (a.tile_cols + 31) / 32 * 32;  // (columns are read 32 at a time)
  const int64_t heads = (int64_t)A.batch * A.kv_heads, tiles = (A.cache + KEYS - 1) / KEYS;
  // keep_q: one wave of two blocks an SM, each an even share of a head's key
  // tiles; else a block for every key tile
  int64_t splits = tiles;
  if (keep_q) {
    splits = std::min(tiles, std::max<int64_t>(1, 2 * (int64_t)ctx->sm_count / heads));
    const int64_t each = (tiles + splits - 1) / splits;
    splits = (tiles + each - 1) / each;
    a.chunk = (int)(each * KEYS);
  } else {
    a.chunk = KEYS;
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
  a.lens = A.lens, a.lse = A.lse, a.acc = A.acc, a.acc_seq = A.acc_seq, a.acc_head = A.acc_head;
  a.c = c, a.decay = (float)A.decay;
  a.rows = A.rows, a.heads = A.heads, a.kv_heads = A.kv_heads, a.cache = A.cache, a.causal = A.causal != 0;
  a.status = ctx->d_status;
  if (A.head_dim <= 64)
    return bf16 ? run<1, true>(ctx, mk, mq, a, heads * splits, keep_q)
                : run<1, false>(ctx, mk, mq, a, heads * splits, keep_q);
  return bf16 ? run<2, true>(ctx, mk, mq, a, heads * splits, keep_q)
              : run<2, false>(ctx, mk, mq, a, heads * splits, keep_q);
}
