// dc_rope.cu -- head norm, rotary positions and the cache append of a batch.
//
// One pass over the fused QKV projection's rows (dc_vgemm's f32 output, or
// 16-bit rows): for a head x of `hd` channels and its weight w
//     y   = x / sqrt(mean(x^2) + eps) * w
//     lo' = lo cos t - hi sin t,  hi' = hi cos t + lo sin t,  (lo, hi) = (y[i], y[i + rot/2])
// queries to their own buffer, keys and values to their cache slots.
//
// Bound by HBM: every element is read once and written once, so nothing is
// staged.  A head belongs to hd/8 neighbouring lanes; a lane holds four
// channels i.. and their partners i + rot/2.., so the rotation needs no
// exchange and the norm one shuffle tree.  The cosines and sines of a row are
// formed once for all its heads: the angle in turns (position x frequency / 2
// pi) in 64 bits, where a position of a million still has 33 bits behind the
// point, its fraction rounded to f32 for sincospi.
#include <math.h>

#include <algorithm>

#include "dc_cache.cuh"

namespace {

using namespace dcc;

constexpr int THREADS = 256;
constexpr int MAX_PAIRS = DC_MAX_ROT / 2;

struct RopeArgs {
  const void* x;
  const int32_t* pos;
  const int64_t* slots;
  const float *wq, *wk;
  void *q, *k, *v;
  int64_t ldx, ld_pos, q_row, q_head, k_seq, k_tok, k_head, v_seq, v_tok, v_head, cache_len, n_slots;
  float eps, inv_hd;
  int rows, heads, kv_heads, hd, rot, tasks, per_block, rows_per_block;
  int* status;
  double turns[MAX_PAIRS];  // frequency of each pair / 2 pi
  uint8_t axis[MAX_PAIRS];
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vec, float (&v)[4]) {
  alignas(16) T h[4];
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = p[i];
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(h) = *reinterpret_cast<const float4*>(p);
  } else {
    *reinterpret_cast<uint2*>(h) = *reinterpret_cast<const uint2*>(p);
  }
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = to_f32(h[i]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, bool vec, const float (&v)[4]) {
  alignas(16) T h[4];
#pragma unroll
  for (int i = 0; i < 4; i++) h[i] = from_f32<T>(v[i]);
  if (!vec) {
#pragma unroll
    for (int i = 0; i < 4; i++) p[i] = h[i];
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(h);
  } else {
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
  }
}

// Blocks along x take rows_per_block rows each, blocks along y per_block of
// their heads (few rows: a block's worth each, so that the call spreads over
// the SMs; many rows: all).  LANES: lanes of a head, a power of two >= hd / 8.
template <typename TI, typename TO, int LANES, bool VEC>
__global__ void __launch_bounds__(THREADS) k_head_norm_rope(const __grid_constant__ RopeArgs a) {
  extern __shared__ float2 cs[];  // rows_per_block x rot/2
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row0 = blockIdx.x * a.rows_per_block;
  const int nrows = min(a.rows_per_block, a.rows - row0);
  const int pairs = a.rot >> 1;
  for (int i = threadIdx.x; i < nrows * pairs; i += THREADS) {
    const int r = i / pairs, p = i - r * pairs;
    const double t = (double)a.pos[a.axis[p] * a.ld_pos + row0 + r] * a.turns[p];
    float s, c;
    sincospif(2.0f * (float)(t - rint(t)), &s, &c);
    cs[i] = make_float2(c, s);
  }
  __syncthreads();
  const int sub = threadIdx.x & (LANES - 1);
  const bool live = sub < (a.hd >> 3);
  const int nrot = a.rot >> 3;
  // this lane's two groups of four channels: a rotated group and its partners,
  // or eight channels that are not rotated
  const bool turn = sub < nrot;
  const int c0 = turn ? 4 * sub : a.rot + 8 * (sub - nrot);
  const int c1 = turn ? c0 + pairs : c0 + 4;
  const int head0 = blockIdx.y * a.per_block;
  const int nheads = min(a.per_block, a.tasks - head0);
  const int total = nrows * nheads;
  // (whole warps stay in the loop: the norm's shuffles name all lanes)
  for (int base = (threadIdx.x >> 5) * (32 / LANES); base < total; base += THREADS / LANES) {
    const int task = base + (threadIdx.x & 31) / LANES;
    const bool on = live && task < total;
    const int r = task / nheads, head = head0 + task - r * nheads;
    const int row = row0 + r;
    const bool is_v = head >= a.heads + a.kv_heads, is_q = head < a.heads;
    float lo[4] = {0, 0, 0, 0}, hi[4] = {0, 0, 0, 0};
    const int d0 = is_v ? 8 * sub : c0, d1 = is_v ? 8 * sub + 4 : c1;
    if (on) {
      const TI* src = (const TI*)a.x + (int64_t)row * a.ldx + (int64_t)head * a.hd;
      load4<TI>(src + d0, VEC, lo);
      load4<TI>(src + d1, VEC, hi);
    }
    const float* w = is_q ? a.wq : a.wk;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) ss = fmaf(lo[i], lo[i], fmaf(hi[i], hi[i], ss));
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
    if (!on) continue;
    TO* dst;
    if (is_q) {
      dst = (TO*)a.q + (int64_t)row * a.q_row + (int64_t)head * a.q_head;
    } else {
      const int64_t slot = a.slots ? a.slots[row] : row;
      if (slot < 0) continue;
      if (slot >= a.n_slots) {
        atomicOr(a.status, DC_ST_BOUNDS);
        continue;
      }
      const int64_t seq = a.n_slots == a.cache_len ? 0 : slot / a.cache_len;
      const int64_t tok = slot - seq * a.cache_len;
      dst = is_v ? (TO*)a.v + seq * a.v_seq + tok * a.v_tok + (head - a.heads - a.kv_heads) * a.v_head
                 : (TO*)a.k + seq * a.k_seq + tok * a.k_tok + (head - a.heads) * a.k_head;
    }
    if (!is_v) {
      if (w) {
        const float inv = __frsqrt_rn(fmaf(ss, a.inv_hd, a.eps));
#pragma unroll
        for (int i = 0; i < 4; i++) {
          lo[i] = lo[i] * inv * __ldg(w + d0 + i);
          hi[i] = hi[i] * inv * __ldg(w + d1 + i);
        }
      }
      if (turn) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float2 t = cs[r * pairs + d0 + i];
          const float l = lo[i], h = hi[i];
          lo[i] = l * t.x - h * t.y;
          hi[i] = h * t.x + l * t.y;
        }
      }
    }
    store4<TO>(dst + d0, VEC, lo);
    store4<TO>(dst + d1, VEC, hi);
  }
}

using Kernel = void (*)(const RopeArgs);

template <typename TI, typename TO, bool VEC>
Kernel by_lanes(int lanes) {
  return lanes == 8    ? k_head_norm_rope<TI, TO, 8, VEC>
         : lanes == 16 ? k_head_norm_rope<TI, TO, 16, VEC>
                       : k_head_norm_rope<TI, TO, 32, VEC>;
}
template <typename TI, typename TO>
Kernel by_vec(int lanes, bool vec) {
  return vec ? by_lanes<TI, TO, true>(lanes) : by_lanes<TI, TO, false>(lanes);
}
template <typename TI>
Kernel by_out(int out, int lanes, bool vec) {
  return out == DC_F32   ? by_vec<TI, float>(lanes, vec)
         : out == DC_F16 ? by_vec<TI, __half>(lanes, vec)
                         : by_vec<TI, __nv_bfloat16>(lanes, vec);
}

}  // namespace

extern "C" int dc_head_norm_rope_dev(dc_ctx* ctx, const dc_head_rope* p) {
  if (!ctx || !p) return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: bad arguments");
  const dc_head_rope& A = *p;
  if (A.rows < 0 || A.heads < 0 || A.kv_heads < 0 || A.heads + (int64_t)A.kv_heads < 1 ||
      A.heads + 2 * (int64_t)A.kv_heads > 65535)
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: rows %d, heads %d, kv_heads %d", A.rows, A.heads, A.kv_heads);
  if (A.head_dim < 8 || A.head_dim > DC_MAX_ROT || (A.head_dim & 7) || A.rot < 0 || A.rot > A.head_dim || (A.rot & 7))
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: head_dim %d (8..%d) and rot %d must be multiples of 8",
                   A.head_dim, DC_MAX_ROT, A.rot);
  if (!is_type(A.x_type) || !is_type(A.out_type)) return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: unknown type");
  if (!(A.eps >= 0.0) || !isfinite(A.eps)) return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: eps");
  if (A.axes < 1 || A.axes > DC_MAX_AXES) return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: %d position axes", A.axes);
  const int pairs = A.rot / 2;
  if (!A.inv_freq && pairs && (!(A.theta > 0.0) || !isfinite(A.theta)))
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: theta");
  RopeArgs a;
  int64_t sum = 0;
  for (int i = 0; i < A.axes; i++) {
    if (A.sections[i] < 0) return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: negative section");
    sum += A.sections[i];
  }
  if (sum != pairs)
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: sections sum to %lld, not rot/2 = %d", (long long)sum, pairs);
  if (A.cyclic) {
    for (int i = 1; i < A.axes; i++)
      if (A.sections[i] > 0 && i + A.axes * (A.sections[i] - 1) >= pairs)
        return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: cyclic section %d does not fit rot/2 = %d", i, pairs);
    for (int i = 0; i < pairs; i++) a.axis[i] = i / A.axes < A.sections[i % A.axes] ? i % A.axes : 0;
  } else {
    for (int i = 0, ax = 0, left = A.sections[0]; i < pairs; i++, left--) {
      while (!left) left = A.sections[++ax];
      a.axis[i] = ax;
    }
  }
  if (!A.rows) return DC_OK;
  if (!A.x || !A.pos || (A.heads && !A.q) || (A.kv_heads && (!A.k || !A.v)))
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: null buffer");
  const int64_t width = (int64_t)(A.heads + 2 * A.kv_heads) * A.head_dim;
  if (A.ldx < width || (A.axes > 1 && A.ld_pos < A.rows))
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: ldx %lld is below a row's %lld, or ld_pos below the rows",
                   (long long)A.ldx, (long long)width);
  if (A.kv_heads && (A.cache_seqs < 1 || A.cache_len < 1 || A.cache_seqs > INT64_MAX / A.cache_len ||
                     (!A.slots && A.rows > A.cache_seqs * A.cache_len)))
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: %d rows for a cache of %lld x %lld slots", A.rows,
                   (long long)A.cache_seqs, (long long)A.cache_len);
  const int es_i = elem_size(A.x_type), es_o = elem_size(A.out_type);
  const Span x = span(A.x, es_i, {{A.rows, A.ldx}, {width, 1}});
  const Span q = span(A.heads ? A.q : nullptr, es_o, {{A.rows, A.q_row}, {A.heads, A.q_head}, {A.head_dim, 1}});
  const Span k = span(A.kv_heads ? A.k : nullptr, es_o,
                      {{A.cache_seqs, A.k_seq}, {A.cache_len, A.k_tok}, {A.kv_heads, A.k_head}, {A.head_dim, 1}});
  const Span v = span(A.kv_heads ? A.v : nullptr, es_o,
                      {{A.cache_seqs, A.v_seq}, {A.cache_len, A.v_tok}, {A.kv_heads, A.v_head}, {A.head_dim, 1}});
  if (!q.ok || !k.ok || !v.ok) return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: negative stride");
  // (k and v may be interleaved in one buffer, so only the same address is refused)
  if (x.meets(q) || x.meets(k) || x.meets(v) || q.meets(k) || q.meets(v) || (k.hi && k.lo == v.lo))
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: an output overlaps x or another output");
  DeviceGuard g;
  if (int rc = g.enter(ctx)) return rc;

  constexpr double inv_2pi = 0.15915494309189533577;
  for (int i = 0; i < pairs; i++)
    a.turns[i] = (A.inv_freq ? A.inv_freq[i] : pow(A.theta, -2.0 * i / A.rot)) * inv_2pi;
  a.x = A.x, a.pos = A.pos, a.slots = A.slots, a.wq = A.wq, a.wk = A.wk, a.q = A.q, a.k = A.k, a.v = A.v;
  a.ldx = A.ldx, a.ld_pos = A.ld_pos, a.q_row = A.q_row, a.q_head = A.q_head;
  a.k_seq = A.k_seq, a.k_tok = A.k_tok, a.k_head = A.k_head;
  a.v_seq = A.v_seq, a.v_tok = A.v_tok, a.v_head = A.v_head;
  a.cache_len = A.kv_heads ? A.cache_len : 1, a.n_slots = A.kv_heads ? A.cache_seqs * A.cache_len : 1;
  a.eps = (float)A.eps, a.inv_hd = 1.0f / A.head_dim;
  a.rows = A.rows, a.heads = A.heads, a.kv_heads = A.kv_heads, a.hd = A.head_dim, a.rot = A.rot;
  a.tasks = A.heads + 2 * A.kv_heads;
  a.status = ctx->d_status;
  const int lanes = A.head_dim <= 64 ? 8 : A.head_dim <= 128 ? 16 : 32;
  const int at_once = THREADS / lanes;
  // rows of a block: as many as its threads form angles for in one step, while
  // the blocks still cover every SM a few times
  int rpb = pairs ? std::min(8, std::max(1, THREADS / pairs)) : 8;
  while (rpb > 1 && A.rows / rpb < 4 * ctx->sm_count) rpb >>= 1;
  a.rows_per_block = rpb;
  const int blocks = (int)(((int64_t)A.rows + rpb - 1) / rpb);
  a.per_block = blocks < 2 * ctx->sm_count ? std::min(a.tasks, at_once) : a.tasks;
  const bool vec = aligned(A.x, es_i, 4 * es_i, {A.ldx}) &&
                   (!A.heads || aligned(A.q, es_o, 4 * es_o, {A.q_row, A.q_head})) &&
                   (!A.kv_heads || (aligned(A.k, es_o, 4 * es_o, {A.k_seq, A.k_tok, A.k_head}) &&
                                    aligned(A.v, es_o, 4 * es_o, {A.v_seq, A.v_tok, A.v_head})));
  Kernel kern = A.x_type == DC_F32   ? by_out<float>(A.out_type, lanes, vec)
                : A.x_type == DC_F16 ? by_out<__half>(A.out_type, lanes, vec)
                                     : by_out<__nv_bfloat16>(A.out_type, lanes, vec);
  return launch(ctx, kern, dim3(blocks, (a.tasks + a.per_block - 1) / a.per_block), THREADS, rpb * pairs * 8, 1, a);
}
