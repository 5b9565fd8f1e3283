// dc_prefix.cu -- attention of a batch over a shared prefix and its own keys.
//
//   x_j = scale * q . k_j,  out = sum_j exp(x_j) v_j / sum_j exp(x_j),  lse = log(sum_j exp(x_j))
//
// over the prefix's tokens and the row's own.  The sum splits by keys: a part
// with maximum m and sums l = sum 2^(c x - m), o = sum 2^(c x - m) v (c = log2 e)
// joins another after both are scaled to the larger maximum.  Three kernels:
//   * k_shared: the rows of all sequences that use one key/value head, 128 or 256
//     a block, against a range of the prefix: one reading of its keys and values
//     for the whole batch;
//   * k_own: a sequence's rows that use one head against a range of its own keys
//     (and a batch's few rows against the prefix);
//   * k_join: the parts of a row, and its last tokens (below).
//
// A running maximum is raised only when a row's has grown by more than 2^8; until
// then o needs no rescaling.  For bf16 the row's probabilities then lie below 2^8, as
// exact there as below 1.  f16 ends at 2^16 and has no normal numbers below 2^-14, so
// there they are formed 2^7 larger, up to 2^15: what is lost of a key far below the
// maximum is at most 2^-32 of it (2^-25 unshifted, and then a few hundred keys 2^-26
// below a dominant one vanished from out, though not from lse).  Parts are stored
// without that factor.
//
// An exponent is c x - m with m = c times the maximum, one multiply-add; the rounding
// of m then shifts all of a row's alike.  Where the maximum is so far from 0 that this
// would show (FAR), and in k_own, which has instructions to spare, it is c times the
// difference to the maximum: with scores of 10^9 and more the product's rounding alone
// passed what f32 exponents hold, and finite scores gave NaN.
//
// Rows of one sequence may see different last tokens (rows > 1).  k_own takes
// only the tokens that all rows see; the up to rows - 1 behind them go to k_join,
// in f32, so a masked value never meets a zero probability in a product (0 x
// NaN).  Value rows behind the last token are zeroed in shared memory for the
// same reason.
//
// k_own does not read what k_shared writes, so it starts as k_shared's blocks
// end: it is launched as its dependent, k_shared releases it only behind its own
// wait for earlier kernels, and one block of k_own waits for k_shared at its end,
// so that k_join, which waits for k_own, finds both complete.
//
// Every wait on a barrier is bounded (dc_ptx.cuh); a block whose wait gives up
// waits for the copies and products that it has in flight (bounded as well) and ends,
// its part without weight, and dc_sync reports it.
#include <algorithm>
#include <type_traits>

#include "dc_cache.cuh"
#include "dc_ring.h"
#include "dc_umma.cuh"

namespace {

using namespace dcc;
using dcu::F2;

constexpr int MAX_ROWS = 16;
constexpr float LN2 = 0.6931471805599453f;
constexpr float RAISE = 8.0f;  // growth of a row's maximum (in powers of two) that rescales it
constexpr float FAR = 4096.0f;  // of a maximum times c
// Powers of two by which f16 probabilities are larger, and the factor that takes it back.
template <bool BF16>
constexpr float UP = BF16 ? 0.0f : 7.0f;
template <bool BF16>
constexpr float DOWN = BF16 ? 1.0f : 0.0078125f;

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
  int few_blocks;    // blocks of k_own that take the prefix
  int64_t own_base;  // first own part
  int* status;
};

// Place of row g of a head's rows (own: of one sequence; else of the batch) in q.
__device__ __forceinline__ int64_t q_place(const PaArgs& a, int h, int g, int seq) {
  const int rr = g / a.group;
  const int b = seq >= 0 ? seq : rr / a.rows, r = seq >= 0 ? rr : rr - b * a.rows;
  return b * a.q_seq + r * a.q_row + (int64_t)(h * a.group + g - rr * a.group) * a.q_head;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t r;
  if (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
  else
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(a), "f"(b));
  return r;
}

// A wait of a whole warp for two barriers at once.
__device__ __forceinline__ bool warp_wait2(uint64_t* x, uint32_t px, uint64_t* y, uint32_t py, int* status) {
  const bool odd = threadIdx.x & 1;
  return dcu::warp_wait_each(odd ? y : x, odd ? py : px, status);
}

// ---- the shared prefix ----------------------------------------------------------
// Two groups of four warps take the softmax of a 128 x 128 tile of scores, a
// thread a query row (TMEM lane); one more warp streams 128-key tiles through a
// ring by TMA, another issues the products
//   S = Q K^T (128 x 128, f32 in TMEM),  O += P V (128 x hd in TMEM)
// with P rounded to the keys' type.  With two tiles of rows each group has its
// own and both use each tile of keys; a tile of rows that is left over has a block
// whose groups take every other tile of keys and join their parts.  One group's softmax runs under the other's products.
//
// One block an SM (224 KB, all 512 TMEM columns).  Heads up to 64 wide leave room
// for P beside S: the next scores are formed as soon as these have been read.
// Wider ones have P written over S, and the next scores wait for the product.
// Either way P goes out in two halves, so that the product starts on the first.
//
// Per 128 x 128 tile and SM the exponential unit needs 1024 cycles, the products 500
// + 500, shared memory 512 + 256 for their operands and 256 for the copies: with
// 64-key tiles in two smaller blocks an SM the operands and copies alone took 1536.
// Measured: 76 us for 256 rows of each of 8 heads on 65536 keys of 128 channels
// (0.9 PFLOP/s, 3.5 TB/s; with the join), about 3700 cycles for a tile of both groups.
// Neither unit is what it waits for (the exponential unit is busy 37% of the time, at
// 64 channels 51%; the tensor pipe 43%): with no exponentials and an eighth of the
// products it still takes 60.  That is a group's chain of score, load, maximum,
// probabilities, store and product, which two groups fill only in part.  Twice the
// warps a group, rolled loops, the maximum of the tile before, a forced
// order of the groups and an issuing warp for each kind of product gave nothing or
// lost; scores of 64 keys, two buffers a group, one being formed under the other's
// softmax, took 106 us for 64 sequences over 65536 keys where this takes 100 (and 53
// for 56 on 24 x 5 drafts of 64 channels); there is no TMEM for a third group.  (What
// is compared here was measured before double waits ordered the warp's memory and far
// scores had their own form: 100 us are 102 now, 56.5 are 57.7, and 28.4, of 32
// sequences over 8192 keys, 29.2.)
constexpr int ROWS = 128;  // query rows of a group: the MMA's M
constexpr int KEYS = 128;  // keys of a tile
constexpr int SH_THREADS = 384;
// (the oldest warps: when the softmax's many instructions compete with theirs for
// a scheduler, theirs go first)
constexpr int MMA_WARP = 0, TMA_WARP = 1, EXP_WARP = 4;

template <int NP>
struct Shared {
  static constexpr int WIDTH = 64 * NP;  // head_dim, padded to panels
  static constexpr int PANEL = 128 * 128;
  static constexpr int TILE = NP * PANEL;
  static constexpr int STAGES = NP == 2 ? 5 : 8;
  static constexpr int BARS = 2 * STAGES + 13;
  static constexpr int SMEM = (2 + STAGES) * TILE + BARS * 8 + 8;  // (and a slot for the TMEM address)
  // TMEM columns of group g: scores, O, probabilities
  static constexpr bool APART = NP == 1;  // probabilities beside the scores
  // Every so many pairs of exponentials one on the multiply-add pipe.  64 sequences
  // over 65536 keys: 100 us with one in eight, 103 with one in four, and before
  // the waits were shortened 104 and 114 with none.  At 64 channels a head none
  // and one in eight take the same.
  static constexpr int FMA_EVERY = NP == 2 ? 8 : 1 << 20;
  static constexpr uint32_t s_col(int g) { return g * 128; }
  static constexpr uint32_t o_col(int g) { return 256 + g * WIDTH; }
  static constexpr uint32_t p_col(int g) { return APART ? 384 + g * 64 : s_col(g); }
};

template <int NP, bool BF16>
__global__ void __launch_bounds__(SH_THREADS, 1)
    k_shared(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
             const __grid_constant__ PaArgs a) {
  using C = Shared<NP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* ring = smem + 2 * C::TILE;
  uint64_t* full = (uint64_t*)(ring + C::STAGES * C::TILE);
  uint64_t* empty = full + C::STAGES;
  uint64_t* s_full = empty + C::STAGES;  // [2] a group's scores are in TMEM
  uint64_t* s_free = s_full + 2;         // [2] and have been read (APART)
  uint64_t* p_ready = s_free + 2;        // [2 x 2] half of its probabilities are in TMEM
  uint64_t* o_done = p_ready + 4;        // [2] its O holds the tile
  uint64_t* q_ready = o_done + 2;        // [2]
  uint64_t* idle = q_ready + 2;          // all products that were issued are complete
  uint32_t* slot = (uint32_t*)(full + C::BARS);

  const int warp = dcu::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // this block's rows and keys; blocks of the same keys are neighbours and read
  // them out of L2
  const int pairs = (a.pre_m + 1) / 2;
  const int pair = blockIdx.x % pairs, t = blockIdx.x / pairs;
  const int h = t % a.kv_heads, split = t / a.kv_heads;
  const int k0 = split * a.pre_chunk, k1 = min(a.prefix, k0 + a.pre_chunk);
  const int n = (k1 - k0 + KEYS - 1) / KEYS;
  const bool two = 2 * pair + 1 < a.pre_m;  // two tiles of rows
  // tiles of keys: all for both groups, or every other
  const int count0 = two ? n : (n + 1) / 2, count1 = two ? n : n / 2;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; i++) {
      dcp::mbar_init(&full[i], 1);
      dcp::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      dcp::mbar_init(&s_full[i], 1);
      dcp::mbar_init(&s_free[i], 4);
      dcp::mbar_init(&p_ready[2 * i], 4);
      dcp::mbar_init(&p_ready[2 * i + 1], 4);
      dcp::mbar_init(&o_done[i], 1);
      dcp::mbar_init(&q_ready[i], 4);
    }
    dcp::mbar_init(idle, 1);
    dcp::mbar_fence_init();
  }
  if (warp == MMA_WARP) dcu::alloc(slot, 512);
  dcu::fence_before();
  __syncthreads();
  dcu::fence_after();
  const uint32_t tmem = dcu::uniform(*slot);
  // (only now: a dependent that takes TMEM before its own wait must not take
  // what a block of this grid still has to get)
  asm volatile("griddepcontrol.launch_dependents;");

  // Place of tile i's keys and values in the ring's order, the order of first use:
  // K0 V0 K1 V1 .. where both groups use each tile, else K0 K1 V0 K2 V1 K3 ..
  auto place_k = [&](int i) { return two ? 2 * i : i ? 2 * i - 1 : 0; };
  auto place_v = [&](int i) { return two ? 2 * i + 1 : i + 1 < n ? 2 * i + 2 : 2 * n - 1; };

  if (warp == TMA_WARP) {
    if (lane == 0) {
      // ---- copies
      int issued = 0;
      for (int s = 0; s < 2 * n; s++, issued++) {
        const int st = s % C::STAGES;
        if (s >= C::STAGES && !dcp::mbar_wait(&empty[st], ((s / C::STAGES) & 1) ^ 1, a.status)) break;
        const bool is_k = two ? !(s & 1) : s == 0 || ((s & 1) && s != 2 * n - 1);
        const int tile = two ? s / 2 : s == 0 ? 0 : is_k ? (s + 1) / 2 : s == 2 * n - 1 ? n - 1 : s / 2 - 1;
        dcp::mbar_expect_tx(&full[st], C::TILE);
#pragma unroll
        for (int p = 0; p < NP; p++)
          dcu::tma_load_3d(ring + st * C::TILE + p * C::PANEL, is_k ? &map_k : &map_v, p * 64, h, k0 + tile * KEYS,
                           &full[st]);
      }
      dcr::drain<C::STAGES>(issued, [&](int st, uint32_t par) { dcp::mbar_wait(&full[st], par, a.status); });
    }
  } else if (warp == MMA_WARP) {
    // ---- products, of the groups by turns: that keeps their softmaxes half a
    // tile apart (with a warp for each group they fell into step, and waited
    // for the tensor pipe and the exponential unit at the same times)
    constexpr uint32_t id_s = dcu::idesc(BF16, KEYS, false), id_o = dcu::idesc(BF16, C::WIDTH, true);
    const uint64_t dq = dcu::desc(dcp::smem_u32(sQ), 0);
    const uint64_t dk = dcu::desc(dcp::smem_u32(ring), 0), dv = dcu::desc(dcp::smem_u32(ring), C::PANEL);
    auto scores = [&](int g, int j) {
      const int s = place_k(two ? j : g + 2 * j), st = s % C::STAGES;
      // the scores before have been read; where the probabilities lie over them, those too
      uint64_t* other = j == 0 ? &q_ready[two ? g : 0] : C::APART ? &s_free[g] : &o_done[g];
      if (!warp_wait2(&full[st], (s / C::STAGES) & 1, other, j ? (j - 1) & 1 : 0, a.status)) return false;
      dcu::fence_after();
      const uint64_t k = dk + st * (C::TILE >> 4), q = dq + (two ? g : 0) * (C::TILE >> 4);
      if (dcu::elect()) {
#pragma unroll
        for (int kk = 0; kk < 4 * NP; kk++) {
          const uint32_t off = ((kk >> 2) * C::PANEL + (kk & 3) * 32) >> 4;
          dcu::mma_ss(tmem + C::s_col(g), q + off, k + off, id_s, kk > 0);
        }
        dcu::commit(&s_full[g]);
        if (!two || g) dcu::commit(&empty[st]);
      }
      __syncwarp();
      return true;
    };
    bool ok = scores(0, 0) && (count1 == 0 || scores(1, 0));
    for (int j = 0; j < count0 && ok; j++) {
#pragma unroll
      for (int g = 0; g < 2; g++) {
        const int count = g ? count1 : count0;
        if (!ok || j >= count) continue;
        if (C::APART && j + 1 < count) ok = scores(g, j + 1);
        const int s = place_v(two ? j : g + 2 * j), st = s % C::STAGES;
        const uint64_t v = dv + st * (C::TILE >> 4);
#pragma unroll
        for (int half = 0; half < 2; half++) {
          ok = ok && (half ? dcu::warp_wait(&p_ready[2 * g + 1], j & 1, a.status)
                           : warp_wait2(&p_ready[2 * g], j & 1, &full[st], (s / C::STAGES) & 1, a.status));
          if (!ok) break;
          dcu::fence_after();
          if (dcu::elect()) {
#pragma unroll
            for (int kk = 4 * half; kk < 4 * half + 4; kk++)
              dcu::mma_ts(tmem + C::o_col(g), tmem + C::p_col(g) + kk * 8, v + (kk * 16 * 128 >> 4), id_o, j > 0 || kk > 0);
            if (half) {
              dcu::commit(&o_done[g]);
              if (!two || g) dcu::commit(&empty[st]);
            }
          }
          __syncwarp();
        }
        if (!C::APART && ok && j + 1 < count) ok = scores(g, j + 1);
      }
    }
    // (also where a wait gave up: nothing reads the ring or writes TMEM any more)
    if (dcu::elect()) dcu::commit(idle);
    __syncwarp();
    dcu::warp_wait(idle, 0, a.status);
  } else if (warp >= EXP_WARP) {
    const int g = (warp - EXP_WARP) >> 2, quarter = warp & 3;  // group, TMEM lanes
    const int m = 2 * pair + (two ? g : 0);
    const int nrows = min(ROWS, a.pre_rows - m * ROWS);
    // ---- Q into shared memory: each lane its own row's place, then rows by
    // turns.  (One tile of rows: the first group's warps bring it.)
    if (two || g == 0) {
      const int row = quarter * 32 + lane;
      const int64_t at = row < nrows ? q_place(a, h, row + m * ROWS, -1) : -1;
      constexpr int CH = 8 * NP, PER = 32 / CH;  // 16-byte chunks of a row, rows at once
      const int ch = lane % CH;
      uint8_t* dst = sQ + g * C::TILE + (ch >> 3) * C::PANEL;
#pragma unroll 8
      for (int it = 0; it < 32 / PER; it++) {
        const int rl = it * PER + lane / CH, r = quarter * 32 + rl;
        const int64_t src = __shfl_sync(~0u, at, rl);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (src >= 0 && ch * 8 < a.hd) v = *reinterpret_cast<const uint4*>((const uint16_t*)a.q + src + ch * 8);
        *reinterpret_cast<uint4*>(dst + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) dcp::mbar_arrive(&q_ready[g]);
    }
    // ---- softmax: this thread's query row is TMEM lane quarter * 32 + lane
    const uint32_t lane_at = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_at = lane_at + C::s_col(g), o_at = lane_at + C::o_col(g), p_at = lane_at + C::p_col(g);
    const bool used = quarter * 32 < nrows;  // (a warp without rows only keeps the barriers going)
    const int count = g ? count1 : count0;
    float mx = -INFINITY, l = 0.0f;  // the maximum in use (scores before c), the sum
    bool ok = true, far = false;     // (far: for a row of this warp)
    for (int j = 0; j < count; j++) {
      if (!dcu::warp_wait(&s_full[g], j & 1, a.status)) { ok = false; break; }
      dcu::fence_after();
      uint32_t s[4][32];
      if (used) {
#pragma unroll
        for (int x = 0; x < 4; x++) dcu::ld32(s_at + x * 32, s[x]);
#pragma unroll
        for (int x = 0; x < 4; x++) dcu::wait_ld(s[x]);
      }
      if (C::APART) {
        dcu::fence_before();
        __syncwarp();
        if (lane == 0) dcp::mbar_arrive(&s_free[g]);
      }
      const int nv = k1 - k0 - (two ? j : g + 2 * j) * KEYS;  // keys of the tile
      F2 c2 = dcu::f2(a.c, a.c), b2 = c2, sum[2] = {dcu::f2(0, 0), dcu::f2(0, 0)};
      if (used) {
        if (nv < KEYS) {
#pragma unroll
          for (int x = 0; x < 4; x++)
#pragma unroll
            for (int y = 0; y < 32; y++)
              if (x * 32 + y >= nv) s[x][y] = __float_as_uint(-INFINITY);
        }
        float m4[4];
#pragma unroll
        for (int x = 0; x < 4; x++) m4[x] = fmaxf(__uint_as_float(s[x][0]), __uint_as_float(s[x][1]));
#pragma unroll
        for (int y = 2; y < 32; y += 2)
#pragma unroll
          for (int x = 0; x < 4; x++) m4[x] = dcu::max3(m4[x], __uint_as_float(s[x][y]), __uint_as_float(s[x][y + 1]));
        const float top = fmaxf(dcu::max3(m4[0], m4[1], m4[2]), m4[3]);
        const auto is_far = [&] { return __any_sync(~0u, mx != -INFINITY && fabsf(mx) * a.c > FAR); };
        if (j == 0) {
          mx = top;
          far = is_far();
        } else if (__any_sync(~0u, top > mx && !((top - mx) * a.c <= RAISE))) {
          // O *= 2^(c (old - new)), once it holds the product of the tile before
          // (the next product needs these probabilities)
          if (C::APART && !dcu::warp_wait(&o_done[g], (j - 1) & 1, a.status)) { ok = false; break; }
          dcu::fence_after();
          const float up = fmaxf(mx, top);
          const float f = mx == -INFINITY ? 0.0f : mx == up ? 1.0f : dcu::ex2((mx - up) * a.c);
          mx = up;
          far = is_far();
          l *= f;
#pragma unroll 1
          for (int col = 0; col < C::WIDTH; col += 16) {
            uint32_t o[16];
            dcu::ld16(o_at + col, o);
            dcu::wait_ld(o);
#pragma unroll
            for (int y = 0; y < 16; y++) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
            dcu::st16(o_at + col, o);
          }
          dcu::wait_st();
        }
        const float m = mx == -INFINITY ? 0.0f : mx;
        float b = fmaf(m, -a.c, UP<BF16>);
        if (far && C::APART) {
          b = UP<BF16>;
#pragma unroll
          for (int x = 0; x < 4; x++)
#pragma unroll
            for (int y = 0; y < 32; y++) s[x][y] = __float_as_uint(__uint_as_float(s[x][y]) - m);
        } else if (far) {
          b = -m;
        }
        b2 = dcu::f2(b, b);
      }
      bool met = true;
      auto exponentials = [&](auto is_far) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
          // (a warp without rows waits too: its arrival belongs to this tile's phase)
          if (C::APART && !used && half == 0 && j > 0) met = dcu::warp_wait(&o_done[g], (j - 1) & 1, a.status);
          if (used) {
#pragma unroll
            for (int x = 2 * half; x < 2 * half + 2; x++) {
              uint32_t p[16];
#pragma unroll
              for (int y = 0; y < 16; y++) {
                // (the sum keeps the unrounded values: lse is exact to f32; P is
                // rounded to the type of the products' operands, half a step each)
                F2 e = dcu::f2(__uint_as_float(s[x][2 * y]), __uint_as_float(s[x][2 * y + 1]));
                if constexpr (decltype(is_far)::value)
                  e = dcu::fma2(dcu::add2(e, b2), c2, dcu::f2(UP<BF16>, UP<BF16>));
                else
                  e = dcu::fma2(e, c2, b2);
                if (y % C::FMA_EVERY == C::FMA_EVERY - 1) {
                  e = dcu::ex2_fma(e);
                } else {
                  const float2 v = dcu::split(e);
                  e = dcu::f2(dcu::ex2(v.x), dcu::ex2(v.y));
                }
                sum[y & 1] = dcu::add2(sum[y & 1], e);
                const float2 v = dcu::split(e);
                p[y] = pack2<BF16>(v.x, v.y);
              }
              // (beside the scores: where the product of the tile before has read the ones there)
              if (C::APART && x == 0 && j > 0) met = dcu::warp_wait(&o_done[g], (j - 1) & 1, a.status);
              dcu::fence_after();
              dcu::st16(p_at + x * 16, p);
            }
            dcu::wait_st();
          }
          dcu::fence_before();
          __syncwarp();
          if (lane == 0) dcp::mbar_arrive(&p_ready[2 * g + half]);
        }
      };
      // (far scores in a loop of their own: taking m off beforehand cost 64 x 65536 3 us in
      // spilled registers; where that costs nothing, at 64 channels, a second loop cost
      // the drafts 2.5)
      if (far && !C::APART)
        exponentials(std::true_type());
      else
        exponentials(std::false_type());
      const float2 both = dcu::split(dcu::add2(sum[0], sum[1]));
      l += both.x + both.y;
      if (!met) { ok = false; break; }
    }
    // ---- the part: through shared memory (the ring, once both groups are done
    // with it), a row to a thread, each then one bulk copy; two groups of one tile
    // of rows join theirs first.  (Stored from registers, 16 bytes a row at a
    // time, this took 2.9 us of a block's 15 at four tiles a block.)
    constexpr int STRIDE = C::WIDTH * 4 + 16;  // rows of neighbouring lanes in different banks
    static_assert(2 * 128 * STRIDE <= C::STAGES * C::TILE, "the ring holds both groups' parts");
    const int row = quarter * 32 + lane;
    uint8_t* mine = ring + (g * 128 + row) * STRIDE;
    ok = ok && count > 0 && used && dcu::warp_wait(&o_done[g], (count - 1) & 1, a.status);
    if (!ok) mx = -INFINITY, l = 0.0f;
    float2 ml = make_float2(mx == -INFINITY ? -INFINITY : mx * a.c, DOWN<BF16> * l);
    dcp::named_sync(1, 256);
    dcu::fence_after();
    // this row, times f, and (join) the second group's, times f_other; a factor of
    // 0 means a part without weight, whose O may be anything
    auto put = [&](bool join, float f, float f_other) {
      const uint8_t* other = mine + 128 * STRIDE;
#pragma unroll 1
      for (int col = 0; col < C::WIDTH; col += 16) {
        uint32_t o[16];
        dcu::ld16(o_at + col, o);
        dcu::wait_ld(o);
#pragma unroll
        for (int y = 0; y < 16; y += 4) {
          float4 v = make_float4(0, 0, 0, 0);
          if (f != 0.0f)
            v = make_float4(f * __uint_as_float(o[y]), f * __uint_as_float(o[y + 1]), f * __uint_as_float(o[y + 2]),
                            f * __uint_as_float(o[y + 3]));
          if (join && f_other != 0.0f) {
            const float4 w = *reinterpret_cast<const float4*>(other + (col + y) * 4);
            v.x = fmaf(f_other, w.x, v.x), v.y = fmaf(f_other, w.y, v.y);
            v.z = fmaf(f_other, w.z, v.z), v.w = fmaf(f_other, w.w, v.w);
          }
          *reinterpret_cast<float4*>(mine + (col + y) * 4) = v;
        }
      }
    };
    if (!two) {
      if (g == 1) {
        if (ok) put(false, 1.0f, 0.0f);
        *reinterpret_cast<float2*>(mine + C::WIDTH * 4) = ml;
      }
      dcp::named_sync(1, 256);
    }
    if (two || g == 0) {
      const int64_t part = ((int64_t)split * a.kv_heads + h) * a.pre_rows + m * ROWS + row;
      if (ok) {
        float f = 1.0f, f_other = 0.0f;
        if (!two) {
          const float2 x = *reinterpret_cast<const float2*>(mine + 128 * STRIDE + C::WIDTH * 4);
          const float top = fmaxf(ml.x, x.x), base = top == -INFINITY ? 0.0f : top;
          f = ml.y == 0.0f ? 0.0f : dcu::ex2(ml.x - base);
          f_other = x.y == 0.0f ? 0.0f : dcu::ex2(x.x - base);
          ml = make_float2(top, fmaf(f_other, x.y, f * ml.y));
        }
        put(!two, f * DOWN<BF16>, f_other * DOWN<BF16>);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        if (row < nrows)
          asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(a.part_o + part * C::WIDTH),
                       "r"(dcp::smem_u32(mine)), "r"(C::WIDTH * 4)
                       : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
      }
      if (row < nrows) a.part_ml[part] = ml;
    }
    dcu::fence_before();
  }
  __syncthreads();
  if (warp == MMA_WARP) {
    dcu::fence_after();
    dcu::dealloc(tmem, 512);
  }
}

// ---- each sequence's own keys ----------------------------------------------------
// Up to 16 query rows a block (row, head of the group), mostly four to eight, so
// the work is the reading of keys and values: HBM-bound.  Each of four warps
// streams its own 16-key tiles (TMA, three in flight, 24 KB a warp: 192 KB an SM
// over two blocks) and keeps its own running maximum, sum and output in registers,
// with 16 x 8 x 16 products (a tcgen05 tile of 128 rows would be empty but for
// these, and its round trips through TMEM cost more than the copies: 41 us
// against HBM's 21 for 64 sequences of up to 1024 tokens).  The warps' results
// join in shared memory.
//
// Where the whole batch has up to FEW_ROWS rows a head, its prefix is taken here
// too, as if it were one sequence's own keys: a tile of 128 rows would be mostly
// empty, and its setup and first products cost more than reading the keys.  8
// key heads of 128 columns, this way and k_shared's, us: 4 rows on 333 keys 5.9
// and 9.6, on 8192 13.0 and 15.4, on 65536 49.9 and 49.1; 32 rows 6.9 and 10.6,
// 15.4 and 17.9, 50.9 and 53.1; 64 rows 8.1 and 10.6, 19.3 and 18.3, 87 and 54.
constexpr int FEW_ROWS = 32;
constexpr int OWN_ROWS = 16;
constexpr int OWN_KEYS = 16;
constexpr int OWN_WARPS = 4;
constexpr int OWN_STAGES = 3;
constexpr int OWN_STEP = OWN_KEYS * OWN_WARPS;

template <int NP>
struct Own {
  static constexpr int WIDTH = 64 * NP;
  static constexpr int PANEL = OWN_KEYS * 128;
  static constexpr int TILE = NP * PANEL;
  static constexpr int WARP = OWN_STAGES * 2 * TILE;  // a warp's ring
  static constexpr int SMEM = OWN_WARPS * WARP + 128;
  static_assert(WARP >= OWN_ROWS * (WIDTH + 4) * 4, "the warps' results are joined in their rings");
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
        "%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// `behind`: launched behind k_shared, whose end it waits for last.
template <int NP, bool BF16>
__global__ void __launch_bounds__(OWN_WARPS * 32, 2)
    k_own(const __grid_constant__ CUtensorMap map_kp, const __grid_constant__ CUtensorMap map_vp,
          const __grid_constant__ CUtensorMap map_ko, const __grid_constant__ CUtensorMap map_vo,
          const __grid_constant__ PaArgs a, const int behind) {
  using C = Own<NP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = (uint64_t*)(smem + OWN_WARPS * C::WARP);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (!behind) asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const bool pre = (int)blockIdx.x < a.few_blocks;
  const int row_tiles = pre ? a.pre_m : a.own_m, splits = pre ? a.pre_splits : a.own_splits;
  int t = blockIdx.x - (pre ? 0 : a.few_blocks);
  const int m = t % row_tiles;
  t /= row_tiles;
  int split, h, seq = -1, k0, k1, rows;
  int64_t part;
  if (pre) {
    h = t % a.kv_heads, split = t / a.kv_heads;
    k0 = split * a.pre_chunk, k1 = min(a.prefix, k0 + a.pre_chunk);
    rows = a.pre_rows;
    part = (int64_t)t * rows;
  } else {
    split = t % splits;
    const int bh = t / splits;
    h = bh % a.kv_heads, seq = bh / a.kv_heads;
    // tokens that all rows see (a length far below 0 is 0 before anything is taken off it)
    const int seen = max(0, max(0, min(a.lens[seq], a.own_max)) - (a.rows - 1));
    k0 = split * a.own_chunk, k1 = min(seen, k0 + a.own_chunk);
    rows = a.own_rows;
    part = a.own_base + (int64_t)t * rows;
  }
  const int nrows = min(OWN_ROWS, rows - m * OWN_ROWS);
  part += m * OWN_ROWS;
  const CUtensorMap *map_k = pre ? &map_kp : &map_ko, *map_v = pre ? &map_vp : &map_vo;
  if (k1 <= k0) {
    if ((int)threadIdx.x < nrows) a.part_ml[part + threadIdx.x] = make_float2(-INFINITY, 0.0f);
  } else {
    uint8_t* ring = smem + warp * C::WARP;
    uint64_t* full = bars + warp * OWN_STAGES;
    const int tiles = (k1 - k0 + OWN_KEYS - 1) / OWN_KEYS, n = (tiles - warp + OWN_WARPS - 1) / OWN_WARPS;
    auto key_of = [&](int i) { return k0 + (i * OWN_WARPS + warp) * OWN_KEYS; };
    auto copy = [&](int i) {
      const int st = i % OWN_STAGES;
      dcp::mbar_expect_tx(&full[st], 2 * C::TILE);
#pragma unroll
      for (int p = 0; p < NP; p++) {
        uint8_t* dst = ring + st * 2 * C::TILE + p * C::PANEL;
        dcu::tma_load_4d(dst, map_k, p * 64, h, key_of(i), pre ? 0 : seq, &full[st]);
        dcu::tma_load_4d(dst + C::TILE, map_v, p * 64, h, key_of(i), pre ? 0 : seq, &full[st]);
      }
    };
    if (lane == 0) {
      for (int i = 0; i < OWN_STAGES; i++) dcp::mbar_init(&full[i], 1);
      dcp::mbar_fence_init();
      for (int i = 0; i < min(n, OWN_STAGES); i++) copy(i);
    }
    __syncwarp();
    // Q fragments: rows lane / 4 and + 8, channels 16 x + 2 (lane % 4) and + 8
    uint32_t q[4 * NP][4];
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int row = lane / 4 + 8 * half;
      const uint16_t* src = (const uint16_t*)a.q + (row < nrows ? q_place(a, h, row + m * OWN_ROWS, seq) : 0);
#pragma unroll
      for (int x = 0; x < 4 * NP; x++)
#pragma unroll
        for (int y = 0; y < 2; y++) {
          const int ch = 16 * x + 8 * y + 2 * (lane % 4);
          q[x][half + 2 * y] = row < nrows && ch < a.hd ? *reinterpret_cast<const uint32_t*>(src + ch) : 0;
        }
    }
    float o[8 * NP][4], mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < 8 * NP; x++)
#pragma unroll
      for (int y = 0; y < 4; y++) o[x][y] = 0.0f;
    int i = 0;
    const int key_k = (lane / 16) * 8 + lane % 8, key_v = ((lane / 8) & 1) * 8 + lane % 8;
    for (; i < n; i++) {
      const int st = i % OWN_STAGES;
      if (!dcu::warp_wait(&full[st], (i / OWN_STAGES) & 1, a.status)) break;
      const int nv = min(OWN_KEYS, k1 - key_of(i));
      const uint32_t k_at = dcp::smem_u32(ring + st * 2 * C::TILE), v_at = k_at + C::TILE;
      float s[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int x = 0; x < 4 * NP; x++) {
        const int ch = 2 * x + ((lane / 8) & 1);
        uint32_t b[4];
        ldmatrix4(b, k_at + (ch >> 3) * C::PANEL + key_k * 128 + (((ch & 7) ^ (key_k & 7)) << 4));
        mma16816<BF16>(s[0], q[x], b[0], b[1]);
        mma16816<BF16>(s[1], q[x], b[2], b[3]);
      }
      if (nv < OWN_KEYS) {
        // value rows behind the last token hold anything: zero them
        for (int j = lane; j < (OWN_KEYS - nv) * 8 * NP; j += 32) {
          const int p = j / ((OWN_KEYS - nv) * 8), rest = j - p * (OWN_KEYS - nv) * 8;
          *reinterpret_cast<uint4*>(ring + st * 2 * C::TILE + C::TILE + p * C::PANEL + nv * 128 + rest * 16) =
              make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int y = 0; y < 4; y++)
            if (8 * x + 2 * (lane % 4) + (y & 1) >= nv) s[x][y] = -INFINITY;
      }
      float top[2] = {fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1])),
                      fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]))};
#pragma unroll
      for (int y = 0; y < 2; y++) {
        top[y] = fmaxf(top[y], __shfl_xor_sync(~0u, top[y], 1));
        top[y] = fmaxf(top[y], __shfl_xor_sync(~0u, top[y], 2));
      }
      bool raise = false;
#pragma unroll
      for (int y = 0; y < 2; y++) raise |= top[y] > mx[y] && !((top[y] - mx[y]) * a.c <= RAISE);
      if (__any_sync(~0u, raise)) {
        float f[2];
#pragma unroll
        for (int y = 0; y < 2; y++) {
          const float up = fmaxf(mx[y], top[y]);
          f[y] = mx[y] == -INFINITY ? 0.0f : mx[y] == up ? 1.0f : dcu::ex2((mx[y] - up) * a.c);
          mx[y] = up;
          l[y] *= f[y];
        }
        if (i > 0) {
#pragma unroll
          for (int x = 0; x < 8 * NP; x++)
#pragma unroll
            for (int y = 0; y < 4; y++) o[x][y] *= f[y >> 1];
        }
      }
      const float m[2] = {mx[0] == -INFINITY ? 0.0f : mx[0], mx[1] == -INFINITY ? 0.0f : mx[1]};
      float e[2][4];
#pragma unroll
      for (int x = 0; x < 2; x++)
#pragma unroll
        for (int y = 0; y < 4; y++) {
          e[x][y] = dcu::ex2(fmaf(s[x][y] - m[y >> 1], a.c, UP<BF16>));
          l[y >> 1] += e[x][y];
        }
      const uint32_t p[4] = {pack2<BF16>(e[0][0], e[0][1]), pack2<BF16>(e[0][2], e[0][3]), pack2<BF16>(e[1][0], e[1][1]),
                             pack2<BF16>(e[1][2], e[1][3])};
#pragma unroll
      for (int x = 0; x < 4 * NP; x++) {
        const int ch = 2 * x + lane / 16;
        uint32_t b[4];
        ldmatrix4_t(b, v_at + (ch >> 3) * C::PANEL + key_v * 128 + (((ch & 7) ^ (key_v & 7)) << 4));
        mma16816<BF16>(o[2 * x], p, b[0], b[1]);
        mma16816<BF16>(o[2 * x + 1], p, b[2], b[3]);
      }
      __syncwarp();
      if (lane == 0 && i + OWN_STAGES < n) copy(i + OWN_STAGES);
    }
    if (i < n) {  // (given up)
      dcr::drain_own<OWN_STAGES>(i, n, [&](int st, uint32_t par) { dcp::mbar_wait(&full[st], par, a.status); });
#pragma unroll
      for (int y = 0; y < 2; y++) mx[y] = -INFINITY, l[y] = 0.0f;
    }
    // ---- the warps' results
    float* mine = (float*)ring;  // 16 rows of WIDTH + 4 floats (the rows of a fragment in different banks)
#pragma unroll
    for (int y = 0; y < 2; y++) {
      l[y] += __shfl_xor_sync(~0u, l[y], 1);
      l[y] += __shfl_xor_sync(~0u, l[y], 2);
      const int row = lane / 4 + 8 * y;
      if (lane % 4 == 0)
        *reinterpret_cast<float2*>(mine + row * (C::WIDTH + 4) + C::WIDTH) =
            make_float2(mx[y] == -INFINITY ? -INFINITY : mx[y] * a.c, DOWN<BF16> * l[y]);
#pragma unroll
      for (int x = 0; x < 8 * NP; x++)
        *reinterpret_cast<float2*>(mine + row * (C::WIDTH + 4) + 8 * x + 2 * (lane % 4)) =
            make_float2(DOWN<BF16> * o[x][2 * y], DOWN<BF16> * o[x][2 * y + 1]);
    }
    __syncthreads();
    for (int j = threadIdx.x; j < nrows * (C::WIDTH / 4); j += OWN_WARPS * 32) {
      const int row = j / (C::WIDTH / 4), col = (j - row * (C::WIDTH / 4)) * 4;
      const float* r = (const float*)smem + row * (C::WIDTH + 4);
      float2 ml[OWN_WARPS];
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < OWN_WARPS; w++) {
        ml[w] = *reinterpret_cast<const float2*>(r + w * (C::WARP / 4) + C::WIDTH);
        top = fmaxf(top, ml[w].x);
      }
      const float base = top == -INFINITY ? 0.0f : top;
      float4 sum = make_float4(0, 0, 0, 0);
      float z = 0.0f;
#pragma unroll
      for (int w = 0; w < OWN_WARPS; w++) {
        const float f = ml[w].y == 0.0f ? 0.0f : dcu::ex2(ml[w].x - base);
        const float4 v = *reinterpret_cast<const float4*>(r + w * (C::WARP / 4) + col);
        z = fmaf(f, ml[w].y, z);
        sum.x = fmaf(f, v.x, sum.x), sum.y = fmaf(f, v.y, sum.y), sum.z = fmaf(f, v.z, sum.z), sum.w = fmaf(f, v.w, sum.w);
      }
      *reinterpret_cast<float4*>(a.part_o + (part + row) * C::WIDTH + col) = sum;
      if (col == 0) a.part_ml[part + row] = make_float2(top, z);
    }
  }
  if (behind && blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- joining the parts ------------------------------------------------------------
// One warp per (sequence, row, query head): joins the parts of its row, eight
// in flight, and scores the own tokens behind those that all rows see.  A lane
// holds WIDTH / 32 channels.
//
// Latency bounds it (a few hundred KB to 12 MB out of L2), so what does not hang
// together is read at once: the last tokens before the parts are complete
// (`behind`: an own kernel before this one has seen to it that q, the caches and
// lens are), the first parts beside their maxima and sums.
template <typename T, int E>
__device__ __forceinline__ void load_f32(const T* src, float (&v)[E]) {  // aligned to its E values
  uint32_t raw[E / 2];
  if constexpr (E == 4) {
    const uint2 x = *reinterpret_cast<const uint2*>(src);
    raw[0] = x.x, raw[1] = x.y;
  } else {
    raw[0] = *reinterpret_cast<const uint32_t*>(src);
  }
  const T* t = reinterpret_cast<const T*>(raw);
#pragma unroll
  for (int e = 0; e < E; e++) v[e] = to_f32(t[e]);
}
template <int NP, typename T, typename TO>
__global__ void __launch_bounds__(128) k_join(const __grid_constant__ PaArgs a, const int behind) {
  constexpr int W = 64 * NP, E = W / 32, EARLY = 4;
  asm volatile("griddepcontrol.launch_dependents;");
  if (!behind) asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (id >= (int64_t)a.batch * a.rows * a.heads) return;
  const int head = id % a.heads, br = id / a.heads, r = br % a.rows, b = br / a.rows;
  const int h = head / a.group, g = head - h * a.group;
  // parts: of the prefix's splits, then of the own splits
  const int total = a.pre_splits + a.own_splits;
  const int64_t pre_at = (int64_t)h * a.pre_rows + br * a.group + g, pre_step = (int64_t)a.kv_heads * a.pre_rows;
  const int64_t own_at = a.own_base + (int64_t)(b * a.kv_heads + h) * a.own_splits * a.own_rows + r * a.group + g;
  auto at = [&](int i) {
    return i < a.pre_splits ? pre_at + i * pre_step : own_at + (int64_t)(i - a.pre_splits) * a.own_rows;
  };
  // the tail's scores, lane j that of token j
  int tail0 = 0, tail = 0;
  float sc = -INFINITY, late[EARLY][E];  // (values of the first few)
  const int c0 = lane * E;
  const bool in = c0 < a.hd;  // (all of a lane's channels, or none: hd is a multiple of 8)
  const T* vp = (const T*)a.v_own + b * a.vo_seq + h * a.vo_head;
  if (a.own_max > 0 && r > 0) {
    const int len = max(0, min(a.lens[b], a.own_max));
    tail0 = max(0, len - (a.rows - 1));
    tail = max(0, len - (a.rows - 1 - r) - tail0);
    float q[E] = {};
    if (in) load_f32((const T*)a.q + b * a.q_seq + r * a.q_row + (int64_t)head * a.q_head + c0, q);
    const T* kp = (const T*)a.k_own + b * a.ko_seq + h * a.ko_head;
#pragma unroll
    for (int j = 0; j < EARLY; j++)
      if (in && j < tail) load_f32(vp + (tail0 + j) * a.vo_tok + c0, late[j]);
#pragma unroll 4
    for (int j = 0; j < tail; j++) {
      float s = 0.0f, k[E];
      if (in) {
        load_f32(kp + (tail0 + j) * a.ko_tok + c0, k);
#pragma unroll
        for (int e = 0; e < E; e++) s = fmaf(q[e], k[e], s);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
      if (lane == j) sc = s * a.c;
    }
  }
  if (behind) asm volatile("griddepcontrol.wait;" ::: "memory");
  auto part = [&](int i, float (&v)[E]) {
    const float* o = a.part_o + at(i) * W + c0;
    if constexpr (E == 4) {
      const float4 f = *reinterpret_cast<const float4*>(o);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
      const float2 f = *reinterpret_cast<const float2*>(o);
      v[0] = f.x, v[1] = f.y;
    }
  };
  float first[8][E];  // (those without weight are whatever was there, and left out below)
#pragma unroll
  for (int j = 0; j < 8; j++)
    if (j < total) part(j, first[j]);
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
    const unsigned some = __ballot_sync(~0u, ml.y != 0.0f);
    const int cnt = min(32, total - i0);
    for (int i = 0; i < cnt; i += 8) {
      if (i0 + i > 0) {
#pragma unroll
        for (int j = 0; j < 8; j++)
          if (some >> (i + j) & 1) part(i0 + i + j, first[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float wj = __shfl_sync(~0u, w, i + j);
        if (some >> (i + j) & 1) {
#pragma unroll
          for (int e = 0; e < E; e++) acc[e] = fmaf(wj, first[j][e], acc[e]);
        }
      }
    }
  }
  if (tail > 0) {
    const float w = lane < tail ? dcu::ex2(sc - base) : 0.0f;
    L += w;
#pragma unroll
    for (int j = 0; j < EARLY; j++) {
      const float wj = __shfl_sync(~0u, w, j);
      if (in && j < tail) {
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] = fmaf(wj, late[j][e], acc[e]);
      }
    }
#pragma unroll 4
    for (int j = EARLY; j < tail; j++) {
      const float wj = __shfl_sync(~0u, w, j);
      float v[E];
      if (in) {
        load_f32(vp + (tail0 + j) * a.vo_tok + c0, v);
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] = fmaf(wj, v[e], acc[e]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  TO* out = (TO*)a.out + b * a.out_seq + r * a.out_row + (int64_t)head * a.out_head;
#pragma unroll
  for (int e = 0; e < E; e++) acc[e] = L == 0.0f ? 0.0f : acc[e] * inv;
  if (in) {
    struct alignas(E * sizeof(TO)) Row {
      TO v[E];
    } row;
#pragma unroll
    for (int e = 0; e < E; e++) row.v[e] = from_f32<TO>(acc[e]);
    *reinterpret_cast<Row*>(out + c0) = row;
  }
  if (a.lse && lane == 0) a.lse[id] = L == 0.0f ? -INFINITY : (base + log2f(L)) * LN2;
}

// How a call's keys are split: the splits follow from sizes alone, so that the
// workspace's size is known before the call.
struct Plan {
  int group, pre_rows, pre_m, pre_chunk, pre_splits, own_rows, own_m, own_chunk, own_splits;
  int64_t pre_blocks, own_blocks, own_base, parts;
  int width;
  bool few;  // the prefix goes to k_own
};
// The number of even shares of `tiles` tiles for each of `items`, `slots` blocks
// at a time, that ends first: a block costs `start` tiles beside its own (TMEM,
// Q, the first copy, its parts), a part about an eighth of a tile of joining.
int shares(int64_t items, int64_t tiles, int64_t slots, int64_t start) {
  if (!items) return 1;
  int64_t best = 1, least = INT64_MAX;
  for (int64_t s = 1; s <= std::min(tiles, 2 * slots / items + 1); s++) {
    const int64_t waves = (items * s + slots - 1) / slots;
    const int64_t end = 8 * waves * (start + (tiles + s - 1) / s) + s;
    if (end < least) least = end, best = s;
  }
  return (int)best;
}
Plan make_plan(const dc_prefix_attn& A, int sm_count) {
  Plan p = {};
  p.group = A.heads / A.kv_heads;
  p.width = A.head_dim <= 64 ? 64 : 128;
  auto split = [](int64_t tiles, int shares, int tile, int* chunk) {
    if (!tiles) return *chunk = 0;
    const int64_t each = (tiles + shares - 1) / shares;
    *chunk = (int)(each * tile);
    return (int)((tiles + each - 1) / each);
  };
  p.pre_rows = A.batch * A.rows * p.group;
  p.few = p.pre_rows <= FEW_ROWS;
  const int tile = p.few ? OWN_STEP : KEYS;
  p.pre_m = (p.pre_rows + (p.few ? OWN_ROWS : ROWS) - 1) / (p.few ? OWN_ROWS : ROWS);
  const int64_t tp = (A.prefix + tile - 1) / tile, hp = (int64_t)A.kv_heads * (p.few ? p.pre_m : (p.pre_m + 1) / 2);
  p.pre_splits = split(tp, p.few ? shares(hp, tp, 2 * sm_count, 4) : shares(hp, tp, sm_count, 3), tile, &p.pre_chunk);
  p.own_rows = A.rows * p.group;
  p.own_m = (p.own_rows + OWN_ROWS - 1) / OWN_ROWS;
  const int64_t to = (A.own_max + OWN_STEP - 1) / OWN_STEP, ho = (int64_t)A.batch * A.kv_heads * p.own_m;
  p.own_splits = split(to, shares(ho, to, 2 * sm_count, 4), OWN_STEP, &p.own_chunk);
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
int run(dc_ctx* ctx, const CUtensorMap (&maps)[4], const PaArgs& a, const Plan& p, bool f32_out) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const bool shared = p.pre_blocks && !p.few;
  const int64_t own = p.own_blocks + (p.few ? p.pre_blocks : 0);
  if (shared)
    if (int rc = launch(ctx, k_shared<NP, BF16>, dim3((unsigned)p.pre_blocks), SH_THREADS, Shared<NP>::SMEM, 1, maps[0],
                        maps[1], a))
      return rc;
  if (own)
    if (int rc = launch(ctx, k_own<NP, BF16>, dim3((unsigned)own), OWN_WARPS * 32, Own<NP>::SMEM, 1, maps[0], maps[1],
                        maps[2], maps[3], a, (int)shared))
      return rc;
  const dim3 grid((unsigned)(((int64_t)a.batch * a.rows * a.heads + 3) / 4));
  return f32_out ? launch(ctx, k_join<NP, T, float>, grid, 128, 0, 1, a, (int)(shared || own))
                 : launch(ctx, k_join<NP, T, T>, grid, 128, 0, 1, a, (int)(shared || own));
}

}  // namespace

extern "C" size_t dc_prefix_attention_ws(const dc_ctx* ctx, const dc_prefix_attn* p) {
  if (!ctx) return 0;
  dc_ctx* c = const_cast<dc_ctx*>(ctx);
  c->err.clear();  // (a message tells a refusal from a call that needs nothing)
  if (!p) dc_fail(c, DC_E_INVAL, "prefix_attention: bad arguments");
  if (!p || check(c, *p) || !p->batch) return 0;
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
  const std::initializer_list<Dim> d_out = {
      {A.batch, A.out_seq}, {A.rows, A.out_row}, {A.heads, A.out_head}, {A.head_dim, 1}};
  const Span o = span(A.out, es_o, d_out);
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
  if (!apart(d_out)) return dc_fail(ctx, DC_E_INVAL, "prefix_attention: two elements of out share an address");
  if (over) return dc_fail(ctx, DC_E_INVAL, "prefix_attention: out, lse or ws overlaps another buffer");
  DeviceGuard guard;
  if (int rc = guard.enter(ctx)) return rc;

  const bool bf16 = A.type == DC_BF16;
  CUtensorMap maps[4];
  memset(maps, 0, sizeof maps);
  const uint64_t hd = A.head_dim, kv = A.kv_heads;
  const uint32_t own_box[4] = {64, 1, OWN_KEYS, 1}, box[3] = {64, 1, KEYS};
  bool ok = true;
  if (A.prefix) {
    const uint64_t dims[4] = {hd, kv, (uint64_t)A.prefix, 1};
    const uint64_t sk[3] = {2 * (uint64_t)A.kp_head, 2 * (uint64_t)A.kp_tok, 0};
    const uint64_t sv[3] = {2 * (uint64_t)A.vp_head, 2 * (uint64_t)A.vp_tok, 0};
    const int rank = pl.few ? 4 : 3;  // (k_own takes a sequence's number too)
    ok = dcu::encode(&maps[0], A.k_pre, bf16, rank, dims, sk, pl.few ? own_box : box) &&
         dcu::encode(&maps[1], A.v_pre, bf16, rank, dims, sv, pl.few ? own_box : box);
  }
  if (A.own_max) {
    const uint64_t dims[4] = {hd, kv, (uint64_t)A.own_max, (uint64_t)A.batch};
    const uint64_t sk[3] = {2 * (uint64_t)A.ko_head, 2 * (uint64_t)A.ko_tok, 2 * (uint64_t)A.ko_seq};
    const uint64_t sv[3] = {2 * (uint64_t)A.vo_head, 2 * (uint64_t)A.vo_tok, 2 * (uint64_t)A.vo_seq};
    ok = ok && dcu::encode(&maps[2], A.k_own, bf16, 4, dims, sk, own_box) &&
         dcu::encode(&maps[3], A.v_own, bf16, 4, dims, sv, own_box);
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
  a.own_base = pl.own_base, a.status = ctx->d_status;
  a.few_blocks = pl.few ? (int)pl.pre_blocks : 0;
  if (pl.pre_blocks + pl.own_blocks > INT32_MAX) return dc_fail(ctx, DC_E_INVAL, "prefix_attention: too many blocks");
  const bool f32_out = A.out_type == DC_F32;
  if (pl.width == 64)
    return bf16 ? run<1, true>(ctx, maps, a, pl, f32_out) : run<1, false>(ctx, maps, a, pl, f32_out);
  return bf16 ? run<2, true>(ctx, maps, a, pl, f32_out) : run<2, false>(ctx, maps, a, pl, f32_out);
}
