// dc_prefix.cu -- attention of a batch over a shared prefix and its own keys.
//
//   x_j = scale * q . k_j,  out = sum_j exp(x_j) v_j / sum_j exp(x_j),  lse = log(sum_j exp(x_j))
//
// over the prefix's tokens and the row's own.  The sum splits by keys: a part
// with maximum m and sums l = sum 2^(c x - m), o = sum 2^(c x - m) v (c = log2 e)
// joins another after both are scaled to the larger maximum.  So every block
// takes one key/value head, one range of keys and up to 128 query rows:
//   * prefix blocks: rows are (sequence, row, head of the group) -- all rows of
//     the batch against one reading of the prefix's keys and values;
//   * own blocks: rows are (row, head of the group) of one sequence.
// k_prefix_attn writes each block's (m, l, o); k_prefix_join joins them.
//
// Bound: HBM while a key/value head has up to ~128 rows (a 64-key tile is 32 KB
// at 43 GB/s an SM, 0.75 us, against 0.3 us of products and as much of
// exponentials); the exponential unit and the tensor pipe above that.
//
// k_prefix_attn: warps 0-3 own a TMEM lane (query row) per thread, warp 4
// streams 64-key tiles through a ring by TMA, warp 5 issues the products
//   S = Q K^T (128 x 64, f32 in TMEM, two buffers), O += P V (128 x hd in TMEM)
// with P, rounded to the keys' type, written over S.  Two blocks share an SM, so
// one's softmax runs under the other's products and copies.  The running maximum
// is raised only when a row's has grown by more than 2^8: until then the row's
// P stay below 2^8, exact enough in either type, and O needs no rescaling.
//
// Rows of one own block may see different last tokens (rows > 1).  The blocks
// take only the tokens that all rows see; the up to rows - 1 behind them go to
// k_prefix_join, in f32, so a masked value never meets a zero probability in a
// product (0 x NaN).  Value rows behind the last token are zeroed in shared
// memory for the same reason.
//
// Every wait is bounded (dc_ptx.cuh); a block whose wait gives up ends, and
// dc_sync reports it.
#include <algorithm>

#include "dc_cache.cuh"
#include "dc_umma.cuh"

namespace {

using namespace dcc;

constexpr int ROWS = 128;      // query rows of a block: the MMA's M
constexpr int KEYS = 64;       // keys of a tile
constexpr int THREADS = 192;
constexpr int MAX_ROWS = 16;
constexpr uint32_t TMEM_COLS = 256;
constexpr uint32_t T_O = 128;  // TMEM columns: S buffers at 0 and 64, O from here
constexpr float LN2 = 0.6931471805599453f;
constexpr float RAISE = 8.0f;  // growth of a row's maximum (in powers of two) that rescales it

template <int NP>
struct Cfg {
  static constexpr int WIDTH = 64 * NP;  // head_dim, padded to panels
  static constexpr int Q_PANEL = ROWS * 128;
  static constexpr int KV_PANEL = KEYS * 128;
  static constexpr int TILE = NP * KV_PANEL;
  // 80 KB of ring beside Q's 16 NP KB: two blocks an SM (227 KB)
  static constexpr int STAGES = NP == 2 ? 5 : 10;
  static constexpr int SMEM = NP * Q_PANEL + STAGES * TILE + 256;
};

struct PaArgs {
  const void *q, *k_own, *v_own;
  const int32_t* lens;
  void* out;
  float* lse;
  float* part_o;
  float2* part_ml;
  int64_t q_seq, q_row, q_head, out_seq, out_row, out_head;
  int64_t ko_seq, ko_tok, ko_head, vo_seq, vo_tok, vo_head;
  float c;  // scale * log2 e
  int batch, rows, heads, kv_heads, group, hd, prefix, own_max;
  int pre_rows, pre_m, pre_chunk, pre_splits;  // rows a head, row tiles, keys a split, splits
  int own_rows, own_m, own_chunk, own_splits;
  int pre_blocks;
  int64_t own_base;  // first own part
  int* status;
};

// Bytes of a row of the (128-byte swizzled) Q panel: 16-byte chunk ch of row r.
__device__ __forceinline__ uint32_t swz(int r, int ch) { return (uint32_t)(r * 128 + ((ch ^ (r & 7)) << 4)); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
  else
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
  return r;
}

// A wait of a whole warp: true where every lane's wait was met.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status) {
  return __all_sync(~0u, dcp::mbar_wait(bar, parity, status));
}

// Position of tile i's keys and values in the ring's order K0 K1 V0 K2 V1 ... of n tiles.
__device__ __forceinline__ int seq_k(int i) { return i ? 2 * i - 1 : 0; }
__device__ __forceinline__ int seq_v(int i, int n) { return i + 1 < n ? 2 * i + 2 : 2 * n - 1; }

template <int NP, bool BF16>
__global__ void __launch_bounds__(THREADS, 2)
    k_prefix_attn(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp,
                  const __grid_constant__ CUtensorMap map_ko, const __grid_constant__ CUtensorMap map_vo,
                  const __grid_constant__ PaArgs a) {
  using C = Cfg<NP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* ring = smem + NP * C::Q_PANEL;
  uint64_t* full = (uint64_t*)(ring + C::STAGES * C::TILE);
  uint64_t* empty = full + C::STAGES;
  uint64_t* s_full = empty + C::STAGES;  // [2] scores of a buffer are in TMEM
  uint64_t* p_ready = s_full + 2;        // [2] its probabilities are
  uint64_t* o_done = p_ready + 2;        // O holds tile i
  uint64_t* q_ready = o_done + 1;
  uint32_t* slot = (uint32_t*)(q_ready + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- this block's rows and keys
  const bool own = (int)blockIdx.x >= a.pre_blocks;
  int h, m, seq = 0, k0, k1, nrows;
  int64_t part;  // of row 0 of this block's rows
  if (!own) {
    // row tiles of the same keys are neighbours: they read them out of L2
    m = blockIdx.x % a.pre_m;
    const int t = blockIdx.x / a.pre_m;
    h = t % a.kv_heads;
    const int split = t / a.kv_heads;
    k0 = split * a.pre_chunk;
    k1 = min(a.prefix, k0 + a.pre_chunk);
    nrows = min(ROWS, a.pre_rows - m * ROWS);
    part = (int64_t)t * a.pre_rows + m * ROWS;
  } else {
    int t = blockIdx.x - a.pre_blocks;
    m = t % a.own_m;
    t /= a.own_m;
    const int split = t % a.own_splits, bh = t / a.own_splits;
    h = bh % a.kv_heads;
    seq = bh / a.kv_heads;
    const int n = max(0, min(a.lens[seq], a.own_max) - (a.rows - 1));  // tokens that all rows see
    k0 = split * a.own_chunk;
    k1 = min(n, k0 + a.own_chunk);
    nrows = min(ROWS, a.own_rows - m * ROWS);
    part = a.own_base + (int64_t)t * a.own_rows + m * ROWS;
  }
  if (k1 <= k0) {
    if ((int)threadIdx.x < nrows) a.part_ml[part + threadIdx.x] = make_float2(-INFINITY, 0.0f);
    return;
  }
  const int n = (k1 - k0 + KEYS - 1) / KEYS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; i++) {
      dcp::mbar_init(&full[i], 1);
      dcp::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      dcp::mbar_init(&s_full[i], 1);
      dcp::mbar_init(&p_ready[i], 4);
    }
    dcp::mbar_init(o_done, 1);
    dcp::mbar_init(q_ready, 4);
    dcp::mbar_fence_init();
  }
  if (warp == 5) dcu::alloc(slot, TMEM_COLS);
  dcu::fence_before();
  __syncthreads();
  dcu::fence_after();
  const uint32_t tmem = *slot;
  // (only now: a dependent that takes TMEM before its own wait must not take
  // what a block of this grid still has to get)
  asm volatile("griddepcontrol.launch_dependents;");

  if (warp == 4) {
    if (lane == 0) {
      // ---- copies: a K or V tile for each position of the ring's order
      int issued = 0;
      for (int s = 0; s < 2 * n; s++, issued++) {
        const int st = s % C::STAGES;
        if (s >= C::STAGES && !dcp::mbar_wait(&empty[st], ((s / C::STAGES) & 1) ^ 1, a.status)) break;
        const bool is_k = s == 0 || ((s & 1) && s != 2 * n - 1);
        const int tile = s == 0 ? 0 : is_k ? (s + 1) / 2 : s == 2 * n - 1 ? n - 1 : s / 2 - 1;
        const int key = k0 + tile * KEYS;
        dcp::mbar_expect_tx(&full[st], C::TILE);
#pragma unroll
        for (int p = 0; p < NP; p++) {
          uint8_t* dst = ring + st * C::TILE + p * C::KV_PANEL;
          if (own)
            dcu::tma_load_4d(dst, is_k ? &map_ko : &map_vo, p * 64, h, key, seq, &full[st]);
          else
            dcu::tma_load_3d(dst, is_k ? &map_kp : &map_vp, p * 64, h, key, &full[st]);
        }
      }
      // (given up: what is in flight lands before the block's memory goes away)
      if (issued < 2 * n)
        for (int s = max(0, issued - C::STAGES); s < issued; s++)
          dcp::mbar_wait(&full[s % C::STAGES], (s / C::STAGES) & 1, a.status);
    }
  } else if (warp == 5) {
    if (lane == 0) {
      // ---- products
      constexpr uint32_t id_s = dcu::idesc(BF16, KEYS, false), id_o = dcu::idesc(BF16, C::WIDTH, true);
      const uint32_t q_at = dcp::smem_u32(sQ), ring_at = dcp::smem_u32(ring);
      bool ok = dcp::mbar_wait(q_ready, 0, a.status);
      auto scores = [&](int i) {
        const int s = seq_k(i), st = s % C::STAGES;
        if (!dcp::mbar_wait(&full[st], (s / C::STAGES) & 1, a.status)) return false;
        dcu::fence_after();
#pragma unroll
        for (int kk = 0; kk < 4 * NP; kk++)
          dcu::mma_ss(tmem + (i & 1) * KEYS, dcu::desc(q_at + (kk >> 2) * C::Q_PANEL + (kk & 3) * 32, 0),
                      dcu::desc(ring_at + st * C::TILE + (kk >> 2) * C::KV_PANEL + (kk & 3) * 32, 0), id_s, kk > 0);
        dcu::commit(&empty[st]);
        dcu::commit(&s_full[i & 1]);
        return true;
      };
      ok = ok && scores(0);
      for (int i = 0; i < n && ok; i++) {
        if (i + 1 < n) {
          // scores i + 1 go where the probabilities of i - 1 are read
          if (i > 0) ok = dcp::mbar_wait(o_done, (i - 1) & 1, a.status);
          ok = ok && scores(i + 1);
        }
        ok = ok && dcp::mbar_wait(&p_ready[i & 1], (i >> 1) & 1, a.status);
        const int s = seq_v(i, n), st = s % C::STAGES;
        ok = ok && dcp::mbar_wait(&full[st], (s / C::STAGES) & 1, a.status);
        if (!ok) break;
        dcu::fence_after();
#pragma unroll
        for (int kk = 0; kk < KEYS / 16; kk++)
          dcu::mma_ts(tmem + T_O, tmem + (i & 1) * KEYS + kk * 8,
                      dcu::desc(ring_at + st * C::TILE + kk * 16 * 128, C::KV_PANEL), id_o, i > 0 || kk > 0);
        dcu::commit(&empty[st]);
        dcu::commit(o_done);
      }
    }
  } else {
    // ---- Q into shared memory, 32 rows a warp: lane's own row's place, then
    // rows by turns
    {
      const int row = warp * 32 + lane;
      int64_t at = -1;
      if (row < nrows) {
        const int g = row + m * ROWS, rr = g / a.group;
        const int b = own ? seq : rr / a.rows, r = own ? rr : rr - b * a.rows;
        at = b * a.q_seq + r * a.q_row + (int64_t)(h * a.group + g - rr * a.group) * a.q_head;
      }
      constexpr int CH = 8 * NP, PER = 32 / CH;  // 16-byte chunks of a row, rows at once
      const int ch = lane % CH;
#pragma unroll
      for (int it = 0; it < 32 / PER; it++) {
        const int rl = it * PER + lane / CH;
        const int64_t src = __shfl_sync(~0u, at, rl);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (src >= 0 && ch * 8 < a.hd) v = *reinterpret_cast<const uint4*>((const uint16_t*)a.q + src + ch * 8);
        *reinterpret_cast<uint4*>(sQ + (ch >> 3) * C::Q_PANEL + swz(warp * 32 + rl, ch & 7)) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) dcp::mbar_arrive(q_ready);
    }
    // ---- softmax: this thread's query row is TMEM lane warp * 32 + lane
    const uint32_t lane_at = tmem + ((uint32_t)(warp * 32) << 16);
    const bool used = warp * 32 < nrows;  // (a warp without rows only keeps the barriers going)
    float mx = -INFINITY, l = 0.0f;       // the maximum in use (scores before c), the sum
    bool ok = true;
    for (int i = 0; i < n; i++) {
      if (!warp_wait(&s_full[i & 1], (i >> 1) & 1, a.status)) { ok = false; break; }
      dcu::fence_after();
      const int nv = min(KEYS, k1 - k0 - i * KEYS);
      if (used) {
        uint32_t s0[32], s1[32];
        dcu::ld32(lane_at + (i & 1) * KEYS, s0);
        dcu::ld32(lane_at + (i & 1) * KEYS + 32, s1);
        dcu::wait_ld(s0);
        dcu::wait_ld(s1);
        if (nv < KEYS) {
#pragma unroll
          for (int j = 0; j < 32; j++) {
            if (j >= nv) s0[j] = __float_as_uint(-INFINITY);
            if (j + 32 >= nv) s1[j] = __float_as_uint(-INFINITY);
          }
        }
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; j++) t[j] = fmaxf(__uint_as_float(s0[j]), __uint_as_float(s1[j]));
#pragma unroll
        for (int j = 8; j < 32; j++) t[j & 7] = fmaxf(t[j & 7], fmaxf(__uint_as_float(s0[j]), __uint_as_float(s1[j])));
        const float top = fmaxf(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])), fmaxf(fmaxf(t[4], t[5]), fmaxf(t[6], t[7])));
        if (i == 0) {
          mx = top;
        } else if (__any_sync(~0u, top > mx && !((top - mx) * a.c <= RAISE))) {
          // O *= 2^(c (old - new)) once the product of tile i - 1 is in it
          const float up = fmaxf(mx, top);
          const float f = mx == -INFINITY ? 0.0f : mx == up ? 1.0f : dcu::ex2((mx - up) * a.c);
          mx = up;
          l *= f;
          // (scores i were issued after product i - 2 was done, so this parity
          // can only mean product i - 1)
          if (!warp_wait(o_done, (i - 1) & 1, a.status)) { ok = false; break; }
          dcu::fence_after();
#pragma unroll 1
          for (int col = 0; col < C::WIDTH; col += 32) {
            uint32_t o[32];
            dcu::ld32(lane_at + T_O + col, o);
            dcu::wait_ld(o);
#pragma unroll
            for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
            dcu::st32(lane_at + T_O + col, o);
          }
          dcu::wait_st();
        }
        const float base = mx == -INFINITY ? 0.0f : mx * a.c;
        float ls[4] = {0, 0, 0, 0};
        uint32_t p[32];
#pragma unroll
        for (int j = 0; j < 16; j++) {
          const float e0 = dcu::ex2(fmaf(__uint_as_float(s0[2 * j]), a.c, -base));
          const float e1 = dcu::ex2(fmaf(__uint_as_float(s0[2 * j + 1]), a.c, -base));
          const float e2 = dcu::ex2(fmaf(__uint_as_float(s1[2 * j]), a.c, -base));
          const float e3 = dcu::ex2(fmaf(__uint_as_float(s1[2 * j + 1]), a.c, -base));
          ls[0] += e0, ls[1] += e1, ls[2] += e2, ls[3] += e3;
          // (the sum keeps the unrounded values: lse is exact to f32; P is
          // rounded to the type of the products' operands, half a step each)
          p[j] = pack2<BF16>(e0, e1);
          p[16 + j] = pack2<BF16>(e2, e3);
        }
        l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
        dcu::st32(lane_at + (i & 1) * KEYS, p);
        dcu::wait_st();
      }
      if (own && nv < KEYS) {
        // value rows behind the last token hold anything: zero them
        const int s = seq_v(i, n), st = s % C::STAGES;
        if (!warp_wait(&full[st], (s / C::STAGES) & 1, a.status)) { ok = false; break; }
        uint8_t* v = ring + st * C::TILE;
        for (int j = threadIdx.x; j < (KEYS - nv) * 8 * NP; j += 128) {
          const int p = j / ((KEYS - nv) * 8), rest = j - p * (KEYS - nv) * 8;
          *reinterpret_cast<uint4*>(v + p * C::KV_PANEL + nv * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      dcu::fence_before();
      __syncwarp();
      if (lane == 0) dcp::mbar_arrive(&p_ready[i & 1]);
    }
    // (one product after the other: a parity alone cannot tell n - 1 from n - 3)
    if (ok && used && (n < 2 || warp_wait(o_done, (n - 2) & 1, a.status)) && warp_wait(o_done, (n - 1) & 1, a.status)) {
      dcu::fence_after();
      const int row = warp * 32 + lane;
      float* dst = a.part_o + (part + row) * C::WIDTH;
#pragma unroll 1
      for (int col = 0; col < C::WIDTH; col += 32) {
        uint32_t o[32];
        dcu::ld32(lane_at + T_O + col, o);
        dcu::wait_ld(o);
        if (row < nrows) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<uint4*>(dst + col + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
        }
      }
      if (row < nrows) a.part_ml[part + row] = make_float2(mx == -INFINITY ? -INFINITY : mx * a.c, l);
    }
    dcu::fence_before();
  }
  __syncthreads();
  if (warp == 5) {
    dcu::fence_after();
    dcu::dealloc(tmem, TMEM_COLS);
  }
}

// One warp per (sequence, row, query head): joins the parts of its row, and
// scores the own tokens behind those that all rows see.  A lane holds WIDTH / 32
// channels.
template <int NP, typename T, typename TO>
__global__ void __launch_bounds__(128) k_prefix_join(const __grid_constant__ PaArgs a) {
  constexpr int W = 64 * NP, E = W / 32;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (id >= (int64_t)a.batch * a.rows * a.heads) return;
  const int head = id % a.heads, br = id / a.heads, r = br % a.rows, b = br / a.rows;
  const int h = head / a.group, g = head - h * a.group;
  // parts: prefix splits, then own splits
  const int64_t pre_at = (int64_t)h * a.pre_rows + (int64_t)br * a.group + g, pre_step = (int64_t)a.kv_heads * a.pre_rows;
  const int64_t own_at = a.own_base + (int64_t)(b * a.kv_heads + h) * a.own_splits * a.own_rows + r * a.group + g;
  const int total = a.pre_splits + a.own_splits;
  auto at = [&](int i) {
    return i < a.pre_splits ? pre_at + i * pre_step : own_at + (int64_t)(i - a.pre_splits) * a.own_rows;
  };
  // the tail's scores, lane j that of token j
  int tail0 = 0, tail = 0;
  float sc = -INFINITY;
  const int c0 = lane * E;
  if (a.own_max > 0 && r > 0) {
    const int len = max(0, min(a.lens[b], a.own_max));
    tail0 = max(0, len - (a.rows - 1));
    tail = max(0, len - (a.rows - 1 - r) - tail0);
    float q[E];
    const T* qp = (const T*)a.q + b * a.q_seq + r * a.q_row + (int64_t)head * a.q_head;
#pragma unroll
    for (int e = 0; e < E; e++) q[e] = c0 + e < a.hd ? to_f32(qp[c0 + e]) : 0.0f;
    const T* kp = (const T*)a.k_own + b * a.ko_seq + h * a.ko_head;
#pragma unroll 4
    for (int j = 0; j < tail; j++) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < E; e++)
        if (c0 + e < a.hd) s = fmaf(q[e], to_f32(kp[(tail0 + j) * a.ko_tok + c0 + e]), s);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
      if (lane == j) sc = s * a.c;
    }
  }
  float M = sc;
  for (int i = lane; i < total; i += 32) M = fmaxf(M, a.part_ml[at(i)].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
  const float base = M == -INFINITY ? 0.0f : M;
  float acc[E], L = 0.0f;
#pragma unroll
  for (int e = 0; e < E; e++) acc[e] = 0.0f;
  for (int i0 = 0; i0 < total; i0 += 32) {
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (i0 + lane < total) ml = a.part_ml[at(i0 + lane)];
    // (a part of sum 0 has no O)
    const float w = ml.y == 0.0f ? 0.0f : dcu::ex2(ml.x - base);
    L += w * ml.y;
    const int cnt = min(32, total - i0);
    const unsigned some = __ballot_sync(~0u, ml.y != 0.0f);
#pragma unroll 4
    for (int i = 0; i < cnt; i++) {
      const float wi = __shfl_sync(~0u, w, i);
      if (!(some >> i & 1)) continue;
      const float* o = a.part_o + at(i0 + i) * W + c0;
      if constexpr (E == 4) {
        const float4 f = *reinterpret_cast<const float4*>(o);
        acc[0] = fmaf(wi, f.x, acc[0]), acc[1] = fmaf(wi, f.y, acc[1]);
        acc[2] = fmaf(wi, f.z, acc[2]), acc[3] = fmaf(wi, f.w, acc[3]);
      } else {
        const float2 f = *reinterpret_cast<const float2*>(o);
        acc[0] = fmaf(wi, f.x, acc[0]), acc[1] = fmaf(wi, f.y, acc[1]);
      }
    }
  }
  if (tail > 0) {
    const float w = lane < tail ? dcu::ex2(sc - base) : 0.0f;
    L += w;
    const T* vp = (const T*)a.v_own + b * a.vo_seq + h * a.vo_head;
#pragma unroll 4
    for (int j = 0; j < tail; j++) {
      const float wj = __shfl_sync(~0u, w, j);
#pragma unroll
      for (int e = 0; e < E; e++)
        if (c0 + e < a.hd) acc[e] = fmaf(wj, to_f32(vp[(tail0 + j) * a.vo_tok + c0 + e]), acc[e]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  TO* out = (TO*)a.out + b * a.out_seq + r * a.out_row + (int64_t)head * a.out_head;
#pragma unroll
  for (int e = 0; e < E; e++)
    if (c0 + e < a.hd) out[c0 + e] = from_f32<TO>(L == 0.0f ? 0.0f : acc[e] * inv);
  if (a.lse && lane == 0) a.lse[id] = L == 0.0f ? -INFINITY : (base + log2f(L)) * LN2;
}

// How a call's keys are split: the splits follow from sizes alone, so that the
// workspace's size is known before the call.
struct Plan {
  int group, pre_rows, pre_m, pre_chunk, pre_splits, own_rows, own_m, own_chunk, own_splits;
  int64_t pre_blocks, own_blocks, own_base, parts;
  int width;
};
Plan make_plan(const dc_prefix_attn& A, int sm_count) {
  Plan p = {};
  p.group = A.heads / A.kv_heads;
  p.width = A.head_dim <= 64 ? 64 : 128;
  p.pre_rows = A.batch * A.rows * p.group;
  p.pre_m = (p.pre_rows + ROWS - 1) / ROWS;
  p.own_rows = A.rows * p.group;
  p.own_m = (p.own_rows + ROWS - 1) / ROWS;
  const int64_t tp = (A.prefix + KEYS - 1) / KEYS, to = (A.own_max + KEYS - 1) / KEYS;
  const int64_t hp = (int64_t)A.kv_heads * p.pre_m, ho = (int64_t)A.batch * A.kv_heads * p.own_m;
  // One wave: two blocks an SM.  Tiles a block (own caches count as half full)
  // from the whole work, but not fewer than four, over which a block's start
  // (TMEM, Q, the first copy) is spread.
  const int64_t slots = 2 * (int64_t)sm_count;
  int64_t per = std::max<int64_t>(4, (hp * tp + ho * ((to + 1) / 2) + slots - 1) / slots);
  // (a second wave is not worth starting for a few blocks; where the sequences'
  // own blocks alone are more than one wave, they queue behind the prefix's)
  for (; hp + ho <= slots; per += (per + 7) / 8) {
    const int64_t sp = (tp + per - 1) / per, so = (to + 2 * per - 1) / (2 * per);
    if (hp * sp + ho * so <= slots) break;
  }
  auto split = [](int64_t tiles, int64_t most, int* chunk) {
    if (!tiles) return *chunk = 0;
    int64_t s = (tiles + most - 1) / most;
    const int64_t each = (tiles + s - 1) / s;  // even shares
    *chunk = (int)(each * KEYS);
    return (int)((tiles + each - 1) / each);
  };
  p.pre_splits = split(tp, per, &p.pre_chunk);
  p.own_splits = split(to, 2 * per, &p.own_chunk);
  p.pre_blocks = hp * p.pre_splits;
  p.own_blocks = ho * p.own_splits;
  p.own_base = (int64_t)p.pre_splits * A.kv_heads * p.pre_rows;
  p.parts = p.own_base + (int64_t)A.batch * A.kv_heads * p.own_splits * p.own_rows;
  return p;
}

int check(dc_ctx* ctx, const dc_prefix_attn& A) {
  if (A.batch < 0 || A.rows < 1 || A.rows > MAX_ROWS || A.heads < 1 || A.kv_heads < 1 || A.heads % A.kv_heads)
    return dc_fail(ctx, DC_E_INVAL, "prefix_attention: batch %d, rows %d (1..%d), heads %d of %d", A.batch, A.rows,
                   MAX_ROWS, A.heads, A.kv_heads);
  if (A.head_dim < 8 || A.head_dim > 128 || (A.head_dim & 7))
    return dc_fail(ctx, DC_E_INVAL, "prefix_attention: head_dim %d must be a multiple of 8 up to 128", A.head_dim);
  if (A.prefix < 0 || A.own_max < 0 || A.prefix > (1 << 30) || A.own_max > (1 << 30))
    return dc_fail(ctx, DC_E_INVAL, "prefix_attention: prefix %d, own_max %d", A.prefix, A.own_max);
  if ((int64_t)A.batch * A.rows * A.heads > (1 << 24) || (int64_t)A.batch * A.kv_heads > (1 << 20))
    return dc_fail(ctx, DC_E_INVAL, "prefix_attention: %d x %d rows of %d heads are too many", A.batch, A.rows, A.heads);
  if (!is_half(A.type) || (A.out_type != A.type && A.out_type != DC_F32))
    return dc_fail(ctx, DC_E_INVAL, "prefix_attention: type f16 or bf16, out_type that or f32");
  const float c = (float)(A.scale * 1.4426950408889634);
  if (!(c > 0.0f) || !isfinite(c)) return dc_fail(ctx, DC_E_INVAL, "prefix_attention: scale %g", A.scale);
  return DC_OK;
}

size_t ws_bytes_of(const Plan& p) { return (size_t)p.parts * (p.width * 4 + 8); }

template <int NP, bool BF16>
int run(dc_ctx* ctx, const CUtensorMap (&maps)[4], const PaArgs& a, int64_t blocks, bool f32_out) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  if (blocks)
    if (int rc = launch(ctx, k_prefix_attn<NP, BF16>, dim3((unsigned)blocks), THREADS, Cfg<NP>::SMEM, 1, maps[0],
                        maps[1], maps[2], maps[3], a))
      return rc;
  const dim3 grid((unsigned)(((int64_t)a.batch * a.rows * a.heads + 3) / 4));
  return f32_out ? launch(ctx, k_prefix_join<NP, T, float>, grid, 128, 0, 1, a)
                 : launch(ctx, k_prefix_join<NP, T, T>, grid, 128, 0, 1, a);
}

}  // namespace

extern "C" size_t dc_prefix_attention_ws(const dc_ctx* ctx, const dc_prefix_attn* p) {
  if (!ctx || !p || check(const_cast<dc_ctx*>(ctx), *p) || !p->batch) return 0;
  return ws_bytes_of(make_plan(*p, ctx->sm_count));
}

extern "C" int dc_prefix_attention_dev(dc_ctx* ctx, const dc_prefix_attn* p, void* ws, size_t ws_bytes) {
  if (!ctx || !p) return dc_fail(ctx, DC_E_INVAL, "prefix_attention: bad arguments");
  const dc_prefix_attn& A = *p;
  if (int rc = check(ctx, A)) return rc;
  if (!A.batch) return DC_OK;
  if (!A.q || !A.out || (A.prefix && (!A.k_pre || !A.v_pre)) || (A.own_max && (!A.k_own || !A.v_own || !A.lens)))
    return dc_fail(ctx, DC_E_INVAL, "prefix_attention: null buffer");
  const int es_o = elem_size(A.out_type);
  auto row_ok = [&](const void* p, int es, int64_t seq, int64_t n, int64_t tok, int heads, int64_t head) {
    return aligned(p, es, 16, {{A.batch, seq}, {n, tok}, {heads, head}});
  };
  if (!row_ok(A.q, 2, A.q_seq, A.rows, A.q_row, A.heads, A.q_head) ||
      !row_ok(A.out, es_o, A.out_seq, A.rows, A.out_row, A.heads, A.out_head) ||
      (A.prefix && (!row_ok(A.k_pre, 2, 0, A.prefix, A.kp_tok, A.kv_heads, A.kp_head) ||
                    !row_ok(A.v_pre, 2, 0, A.prefix, A.vp_tok, A.kv_heads, A.vp_head))) ||
      (A.own_max && (!row_ok(A.k_own, 2, A.ko_seq, A.own_max, A.ko_tok, A.kv_heads, A.ko_head) ||
                     !row_ok(A.v_own, 2, A.vo_seq, A.own_max, A.vo_tok, A.kv_heads, A.vo_head))))
    return dc_fail(ctx, DC_E_INVAL, "prefix_attention: q, k, v and out rows must begin on 16-byte boundaries");
  const Plan pl = make_plan(A, ctx->sm_count);
  const size_t need = ws_bytes_of(pl);
  if (need && (!ws || ws_bytes < need || ((uintptr_t)ws & 15)))
    return dc_fail(ctx, DC_E_INVAL, "prefix_attention: workspace of %zu bytes, %zu needed (16-byte aligned)", ws_bytes,
                   need);
  const Span q = span(A.q, 2, {{A.batch, A.q_seq}, {A.rows, A.q_row}, {A.heads, A.q_head}, {A.head_dim, 1}});
  const Span o = span(A.out, es_o, {{A.batch, A.out_seq}, {A.rows, A.out_row}, {A.heads, A.out_head}, {A.head_dim, 1}});
  const Span l = span(A.lse, 4, {{(int64_t)A.batch * A.rows * A.heads, 1}});
  const Span w = span(need ? ws : nullptr, 1, {{(int64_t)need, 1}});
  const Span n = span(A.own_max ? A.lens : nullptr, 4, {{A.batch, 1}});
  const Span in[4] = {
      span(A.prefix ? A.k_pre : nullptr, 2, {{A.prefix, A.kp_tok}, {A.kv_heads, A.kp_head}, {A.head_dim, 1}}),
      span(A.prefix ? A.v_pre : nullptr, 2, {{A.prefix, A.vp_tok}, {A.kv_heads, A.vp_head}, {A.head_dim, 1}}),
      span(A.own_max ? A.k_own : nullptr, 2,
           {{A.batch, A.ko_seq}, {A.own_max, A.ko_tok}, {A.kv_heads, A.ko_head}, {A.head_dim, 1}}),
      span(A.own_max ? A.v_own : nullptr, 2,
           {{A.batch, A.vo_seq}, {A.own_max, A.vo_tok}, {A.kv_heads, A.vo_head}, {A.head_dim, 1}})};
  bool bad = !q.ok || !o.ok, over = o.meets(q) || l.meets(q) || w.meets(q) || o.meets(l) || o.meets(w) || l.meets(w) ||
                                    o.meets(n) || l.meets(n) || w.meets(n);
  for (const Span& s : in) {
    bad |= !s.ok;
    over |= o.meets(s) || l.meets(s) || w.meets(s);
  }
  if (bad) return dc_fail(ctx, DC_E_INVAL, "prefix_attention: negative stride");
  if (over) return dc_fail(ctx, DC_E_INVAL, "prefix_attention: out, lse or ws overlaps another buffer");
  DeviceGuard guard;
  if (int rc = guard.enter(ctx)) return rc;

  const bool bf16 = A.type == DC_BF16;
  CUtensorMap maps[4];
  memset(maps, 0, sizeof maps);
  const uint64_t hd = A.head_dim, kv = A.kv_heads;
  const uint32_t box[4] = {64, 1, KEYS, 1};
  bool ok = true;
  if (A.prefix) {
    const uint64_t dims[3] = {hd, kv, (uint64_t)A.prefix};
    const uint64_t sk[2] = {2 * (uint64_t)A.kp_head, 2 * (uint64_t)A.kp_tok};
    const uint64_t sv[2] = {2 * (uint64_t)A.vp_head, 2 * (uint64_t)A.vp_tok};
    ok = dcu::encode(&maps[0], A.k_pre, bf16, 3, dims, sk, box) && dcu::encode(&maps[1], A.v_pre, bf16, 3, dims, sv, box);
  }
  if (A.own_max) {
    const uint64_t dims[4] = {hd, kv, (uint64_t)A.own_max, (uint64_t)A.batch};
    const uint64_t sk[3] = {2 * (uint64_t)A.ko_head, 2 * (uint64_t)A.ko_tok, 2 * (uint64_t)A.ko_seq};
    const uint64_t sv[3] = {2 * (uint64_t)A.vo_head, 2 * (uint64_t)A.vo_tok, 2 * (uint64_t)A.vo_seq};
    ok = ok && dcu::encode(&maps[2], A.k_own, bf16, 4, dims, sk, box) &&
         dcu::encode(&maps[3], A.v_own, bf16, 4, dims, sv, box);
  }
  if (!ok) return dc_fail(ctx, DC_E_INVAL, "prefix_attention: these k or v strides make no tensor map");

  PaArgs a;
  a.q = A.q, a.k_own = A.k_own, a.v_own = A.v_own, a.lens = A.lens, a.out = A.out, a.lse = A.lse;
  a.part_o = (float*)ws;
  a.part_ml = (float2*)((char*)ws + (size_t)pl.parts * pl.width * 4);
  a.q_seq = A.q_seq, a.q_row = A.q_row, a.q_head = A.q_head;
  a.out_seq = A.out_seq, a.out_row = A.out_row, a.out_head = A.out_head;
  a.ko_seq = A.ko_seq, a.ko_tok = A.ko_tok, a.ko_head = A.ko_head;
  a.vo_seq = A.vo_seq, a.vo_tok = A.vo_tok, a.vo_head = A.vo_head;
  a.c = (float)(A.scale * 1.4426950408889634);
  a.batch = A.batch, a.rows = A.rows, a.heads = A.heads, a.kv_heads = A.kv_heads, a.group = pl.group;
  a.hd = A.head_dim, a.prefix = A.prefix, a.own_max = A.own_max;
  a.pre_rows = pl.pre_rows, a.pre_m = pl.pre_m, a.pre_chunk = pl.pre_chunk, a.pre_splits = pl.pre_splits;
  a.own_rows = pl.own_rows, a.own_m = pl.own_m, a.own_chunk = pl.own_chunk, a.own_splits = pl.own_splits;
  a.pre_blocks = (int)pl.pre_blocks, a.own_base = pl.own_base, a.status = ctx->d_status;
  const int64_t blocks = pl.pre_blocks + pl.own_blocks;
  if (blocks > INT32_MAX) return dc_fail(ctx, DC_E_INVAL, "prefix_attention: too many blocks");
  const bool f32_out = A.out_type == DC_F32;
  if (pl.width == 64)
    return bf16 ? run<1, true>(ctx, maps, a, blocks, f32_out) : run<1, false>(ctx, maps, a, blocks, f32_out);
  return bf16 ? run<2, true>(ctx, maps, a, blocks, f32_out) : run<2, false>(ctx, maps, a, blocks, f32_out);
}
