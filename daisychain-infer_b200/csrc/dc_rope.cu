// dc_rope.cu -- head norm, rotary positions and the cache append of a batch.
//
// One pass over the fused QKV projection's rows (dc_vgemm's f32 output, or
// 16-bit rows): for a head x of `hd` channels and its weight w
//     y   = x / sqrt(mean(x^2) + eps) * w
//     lo' = lo cos t - hi sin t,  hi' = hi cos t + lo sin t,  (lo, hi) = (y[i], y[i + rot/2])
// queries to their own buffer, keys and values to their cache slots.
//
// Every element is read once and written once, so nothing is staged.  A head
// belongs to hd/16 neighbouring lanes (hd/8 where rows are not aligned); a lane holds
// eight (four) channels i.. and their partners i + rot/2.., so the rotation needs no
// exchange and the norm one shuffle tree, and a warp walks a row's heads with
// the lane's angles in registers: the angle in turns (position x frequency / 2
// pi) in 64 bits, where a position of a million still has 33 bits behind the
// point, its fraction rounded to f32 for sincospi.
//
// Measured: 2048 rows of 32 + 2 x 8 heads of 128, f32 to bf16, 23.0 us (75 MB, 3.3
// TB/s); 10007 rows of 32 + 2 x 4 heads of 64, f16, three axes, 28.9 us (103 MB, 3.6
// TB/s); 32 rows 3.2 us.  What keeps it from HBM's rate is how little is in flight,
// and that is this form's choice: three or four heads a lane at 128 registers (the
// f32 variants spill 12 bytes) leave 16 warps an SM, a warp asks for the next item only
// when it is done with one (load, angles, norm, store), items are uneven (a row's
// last one may hold a single step of four and waits as long), and an f32 lane's two
// 16-byte loads each touch half of a sector.  Loads through shared memory by each lane
// (24.7 and 29.7 us where this took 22.7 and 28.6) and a whole row an item (20.0 and
// 33.0) were no better for both; bulk copies into a ring have not been tried.
#include <math.h>

#include <algorithm>

#include "dc_cache.cuh"
#include "dc_umma.cuh"

namespace {

using namespace dcc;
using dcu::F2;
using dcu::f2;
using dcu::fma2;
using dcu::mul2;
using dcu::split;

constexpr int THREADS = 256;
// heads a lane holds at once (32 or 48 registers of raw channels)
template <typename T>
constexpr int MAX_STEPS = sizeof(T) == 4 ? 3 : 4;
constexpr int MAX_PAIRS = DC_MAX_ROT / 2;

struct RopeArgs {
  const void* x;
  const int32_t* pos;
  const int64_t* slots;
  const float *wq, *wk;
  void *q, *k, *v;
  int64_t ldx, ld_pos, q_row, q_head, k_seq, k_tok, k_head, v_seq, v_tok, v_head, cache_len, n_slots;
  float eps, inv_hd;
  int rows, heads, kv_heads, hd, rot, parts, q_parts, steps;
  int64_t items;
  int* status;
  double turns[MAX_PAIRS];  // frequency of each pair / 2 pi
  uint8_t axis[MAX_PAIRS];
};

// G neighbouring channels as they lie in memory (VEC: 16-byte pieces).
template <typename T, int G>
struct alignas(16) Some {
  T v[G];
};
template <bool VEC, int G, typename T>
__device__ __forceinline__ Some<T, G> load(const T* p) {
  Some<T, G> f;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)(G * sizeof(T)) / 16; i++)
      reinterpret_cast<uint4*>(&f)[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < G; i++) f.v[i] = p[i];
  }
  return f;
}
__device__ __forceinline__ F2 pair(const float* p) { return f2(p[0], p[1]); }
__device__ __forceinline__ F2 pair(const __half* p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(p));
  return f2(f.x, f.y);
}
__device__ __forceinline__ F2 pair(const __nv_bfloat16* p) {
  const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
  return f2(f.x, f.y);
}
__device__ __forceinline__ void unpair(float* p, float2 f) { p[0] = f.x, p[1] = f.y; }
__device__ __forceinline__ void unpair(__half* p, float2 f) { *reinterpret_cast<__half2*>(p) = __float22half2_rn(f); }
__device__ __forceinline__ void unpair(__nv_bfloat16* p, float2 f) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __float22bfloat162_rn(f);
}
template <bool VEC, int G, typename T>
__device__ __forceinline__ void store(T* p, const F2 (&x)[G / 2]) {
  Some<T, G> f;
#pragma unroll
  for (int i = 0; i < G / 2; i++) unpair(f.v + 2 * i, split(x[i]));
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)(G * sizeof(T)) / 16; i++)
      reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(&f)[i];
  } else {
#pragma unroll
    for (int i = 0; i < G; i++) p[i] = f.v[i];
  }
}

// A work item is a share of a row's query heads, or of its key and value heads.
// Its warp holds SEGS = 32 / LANES heads side by side, `steps` deep, and loads
// all of them, its angles' positions and its slot before it uses any.  A lane
// holds G channels and their G partners of a head; its angles and weights are
// the same for every head of the item (the segments share the making of the
// angles).  Blocks walk the items; the frequencies lie in shared memory, since
// lanes that read different kernel parameters wait for each other.
template <typename TI, typename TO, int LANES, int G, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) k_head_norm_rope(const __grid_constant__ RopeArgs a) {
  constexpr int SEGS = 32 / LANES, EACH = SEGS >= G ? 1 : G / SEGS;  // angles a lane makes
  constexpr int STEPS = MAX_STEPS<TI>;
  __shared__ double turns[MAX_PAIRS];
  __shared__ int64_t pos_at[MAX_PAIRS];
  const int pairs = a.rot >> 1;
  for (int i = threadIdx.x; i < pairs; i += THREADS) {
    turns[i] = a.turns[i];
    pos_at[i] = a.axis[i] * a.ld_pos;
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, sub = lane & (LANES - 1), seg = lane / LANES;
  const int nrot = a.rot / (2 * G);
  const bool live = sub < a.hd / (2 * G), turn = sub < nrot;
  // this lane's two groups of channels: a rotated group and its partners, or
  // two groups that are not rotated
  const int c0 = turn ? G * sub : a.rot + 2 * G * (sub - nrot);
  const int c1 = turn ? c0 + pairs : c0 + G;
  for (int64_t id = (int64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); id < a.items;
       id += (int64_t)gridDim.x * (THREADS / 32)) {
    const int row = (int)(id / a.parts), part = (int)(id - (int64_t)row * a.parts);
    const bool is_q = part < a.q_parts;
    // heads of the item: from h0 of the queries, or of the keys and then values
    const int h0 = (is_q ? part : part - a.q_parts) * a.steps * SEGS + seg;
    const int heads = is_q ? a.heads : 2 * a.kv_heads;
    const TI* x = (const TI*)a.x + row * a.ldx + (is_q ? 0 : a.heads * a.hd);
    Some<TI, G> lo[STEPS], hi[STEPS];
#pragma unroll
    for (int u = 0; u < STEPS; u++) {
      const int h = h0 + u * SEGS;
      if (u < a.steps && live && h < heads) {
        lo[u] = load<VEC, G>(x + h * a.hd + c0);
        hi[u] = load<VEC, G>(x + h * a.hd + c1);
      }
    }
    int64_t slot = is_q ? 0 : a.slots ? a.slots[row] : row;
    const float* w = is_q ? a.wq : a.wk;
    Some<float, G> wl, wh;
    if (w && live) {
      wl = load<VEC, G>(w + c0);
      wh = load<VEC, G>(w + c1);
    }
    F2 c[G / 2], s[G / 2], ns[G / 2];
    {
      float mc[EACH], ms[EACH];
#pragma unroll
      for (int i = 0; i < EACH; i++) {
        mc[i] = 1.0f, ms[i] = 0.0f;
        const int p = c0 + (seg * EACH + i) % G;
        if (turn) {
          const double t = (double)a.pos[pos_at[p] + row] * turns[p];
          sincospif(2.0f * (float)(t - rint(t)), &ms[i], &mc[i]);
        }
      }
      float ca[G], sa[G];
#pragma unroll
      for (int i = 0; i < G; i++) {
        ca[i] = SEGS == 1 ? mc[i] : __shfl_sync(~0u, mc[i % EACH], sub + i / EACH * LANES);
        sa[i] = SEGS == 1 ? ms[i] : __shfl_sync(~0u, ms[i % EACH], sub + i / EACH * LANES);
      }
#pragma unroll
      for (int i = 0; i < G / 2; i++) {
        c[i] = f2(ca[2 * i], ca[2 * i + 1]);
        s[i] = f2(sa[2 * i], sa[2 * i + 1]);
        ns[i] = f2(-sa[2 * i], -sa[2 * i + 1]);
      }
    }
    TO *at = (TO*)a.q + row * a.q_row, *v_at = nullptr;
    int64_t step = a.q_head;
    if (!is_q) {
      if (slot >= a.n_slots) {
        if (lane == 0) atomicOr(a.status, DC_ST_BOUNDS);
        slot = -1;
      }
      const int64_t seq = a.n_slots == a.cache_len || slot < 0 ? 0 : slot / a.cache_len, tok = slot - seq * a.cache_len;
      at = (TO*)a.k + seq * a.k_seq + tok * a.k_tok;
      v_at = (TO*)a.v + seq * a.v_seq + tok * a.v_tok - a.kv_heads * a.v_head;
      step = a.k_head;
    }
#pragma unroll
    for (int u = 0; u < STEPS; u++) {
      if (u >= a.steps) break;
      const int h = h0 + u * SEGS;
      const bool is_v = !is_q && h >= a.kv_heads;
      F2 x0[G / 2], x1[G / 2];
#pragma unroll
      for (int i = 0; i < G / 2; i++) x0[i] = pair(lo[u].v + 2 * i), x1[i] = pair(hi[u].v + 2 * i);
      if (w) {
        F2 sq = mul2(x0[0], x0[0]);
#pragma unroll
        for (int i = 1; i < G / 2; i++) sq = fma2(x0[i], x0[i], sq);
#pragma unroll
        for (int i = 0; i < G / 2; i++) sq = fma2(x1[i], x1[i], sq);
        const float2 both = split(sq);
        float ss = live ? both.x + both.y : 0.0f;
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
        const float inv = rsqrtf(fmaf(ss, a.inv_hd, a.eps));
        if (!is_v) {
          const F2 inv2 = f2(inv, inv);
#pragma unroll
          for (int i = 0; i < G / 2; i++) {
            x0[i] = mul2(x0[i], mul2(inv2, pair(wl.v + 2 * i)));
            x1[i] = mul2(x1[i], mul2(inv2, pair(wh.v + 2 * i)));
          }
        }
      }
      if (turn && !is_v) {
#pragma unroll
        for (int i = 0; i < G / 2; i++) {
          const F2 l = x0[i], r = x1[i];
          x0[i] = fma2(r, ns[i], mul2(l, c[i]));
          x1[i] = fma2(l, s[i], mul2(r, c[i]));
        }
      }
      if (live && h < heads && slot >= 0) {
        TO* p = is_v ? v_at + h * a.v_head : at + h * step;
        store<VEC, G>(p + c0, x0);
        store<VEC, G>(p + c1, x1);
      }
    }
  }
}

using Kernel = void (*)(const RopeArgs);

// hd <= 64, 128 or 256.  Groups of eight channels where rot and hd are
// multiples of 16 and rows begin on 16-byte boundaries (a quarter fewer
// instructions a channel than groups of four), else of four, one by one.
template <typename TI, typename TO>
Kernel by_size(int hd, bool wide) {
  if (wide)
    return hd <= 64    ? k_head_norm_rope<TI, TO, 4, 8, true>
           : hd <= 128 ? k_head_norm_rope<TI, TO, 8, 8, true>
                       : k_head_norm_rope<TI, TO, 16, 8, true>;
  return hd <= 64    ? k_head_norm_rope<TI, TO, 8, 4, false>
         : hd <= 128 ? k_head_norm_rope<TI, TO, 16, 4, false>
                     : k_head_norm_rope<TI, TO, 32, 4, false>;
}
template <typename TI>
Kernel by_out(int out, int hd, bool wide) {
  return out == DC_F32   ? by_size<TI, float>(hd, wide)
         : out == DC_F16 ? by_size<TI, __half>(hd, wide)
                         : by_size<TI, __nv_bfloat16>(hd, wide);
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
  if ((A.rows > 1 && A.ldx < width) || (A.axes > 1 && A.ld_pos < 0))  // (ld_pos 0: the same positions on all axes)
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: ldx %lld is below a row's %lld, or ld_pos negative",
                   (long long)A.ldx, (long long)width);
  if (A.kv_heads && (A.cache_seqs < 1 || A.cache_len < 1 || A.cache_seqs > INT64_MAX / A.cache_len ||
                     (!A.slots && A.rows > A.cache_seqs * A.cache_len)))
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: %d rows for a cache of %lld x %lld slots", A.rows,
                   (long long)A.cache_seqs, (long long)A.cache_len);
  const int es_i = elem_size(A.x_type), es_o = elem_size(A.out_type);
  const Span x = span(A.x, es_i, {{A.rows, A.ldx}, {width, 1}});
  const std::initializer_list<Dim> dq = {{A.rows, A.q_row}, {A.heads, A.q_head}, {A.head_dim, 1}};
  const std::initializer_list<Dim> dk = {
      {A.cache_seqs, A.k_seq}, {A.cache_len, A.k_tok}, {A.kv_heads, A.k_head}, {A.head_dim, 1}};
  const std::initializer_list<Dim> dv = {
      {A.cache_seqs, A.v_seq}, {A.cache_len, A.v_tok}, {A.kv_heads, A.v_head}, {A.head_dim, 1}};
  const Span q = span(A.heads ? A.q : nullptr, es_o, dq), k = span(A.kv_heads ? A.k : nullptr, es_o, dk),
             v = span(A.kv_heads ? A.v : nullptr, es_o, dv);
  if (!q.ok || !k.ok || !v.ok) return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: negative stride");
  if (!apart(dq) || !apart(dk) || !apart(dv))
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: two elements of q, k or v share an address");
  // (k and v may be interleaved in one buffer)
  if (x.meets(q) || x.meets(k) || x.meets(v) || q.meets(k) || q.meets(v) || !twins_apart(k, v, es_o, dk, dv))
    return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: an output overlaps x or another output");
  const Span in[4] = {span(A.pos, 4, {{A.axes, A.ld_pos}, {A.rows, 1}}), span(A.kv_heads ? A.slots : nullptr, 8, {{A.rows, 1}}),
                      span(A.wq, 4, {{A.head_dim, 1}}), span(A.wk, 4, {{A.head_dim, 1}})};
  for (const Span& i : in)
    if (i.meets(q) || i.meets(k) || i.meets(v))
      return dc_fail(ctx, DC_E_INVAL, "head_norm_rope: an output overlaps pos, slots or a norm's weights");
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
  a.status = ctx->d_status;
  auto row_ok = [](const void* p, int es, std::initializer_list<Dim> dims) { return aligned(p, es, 16, dims); };
  const bool wide = !(A.rot % 16) && !(A.head_dim % 16) && row_ok(A.x, es_i, {{A.rows, A.ldx}}) && row_ok(A.wq, 4, {}) &&
                    row_ok(A.wk, 4, {}) && (!A.heads || row_ok(A.q, es_o, {{A.rows, A.q_row}, {A.heads, A.q_head}})) &&
                    (!A.kv_heads ||
                     (row_ok(A.k, es_o, {{A.cache_seqs, A.k_seq}, {A.cache_len, A.k_tok}, {A.kv_heads, A.k_head}}) &&
                      row_ok(A.v, es_o, {{A.cache_seqs, A.v_seq}, {A.cache_len, A.v_tok}, {A.kv_heads, A.v_head}})));
  // items of a row: as few as the steps allow (each makes the row's angles
  // again), but enough for 32 warps an SM when rows are few
  const int segs = 32 / ((A.head_dim <= 64 ? 8 : A.head_dim <= 128 ? 16 : 32) / (wide ? 2 : 1));
  const int most = A.x_type == DC_F32 ? MAX_STEPS<float> : MAX_STEPS<__half>;
  const int q_deep = (A.heads + segs - 1) / segs, kv_deep = (2 * A.kv_heads + segs - 1) / segs;
  const int64_t want = 32 * (int64_t)ctx->sm_count / A.rows;  // items of a row
  a.steps = (int)std::min<int64_t>(most, std::max<int64_t>(1, (q_deep + kv_deep) / std::max<int64_t>(1, want)));
  a.q_parts = (q_deep + a.steps - 1) / a.steps;
  a.parts = a.q_parts + (kv_deep + a.steps - 1) / a.steps;
  a.items = (int64_t)A.rows * a.parts;
  Kernel kern = A.x_type == DC_F32   ? by_out<float>(A.out_type, A.head_dim, wide)
                : A.x_type == DC_F16 ? by_out<__half>(A.out_type, A.head_dim, wide)
                                     : by_out<__nv_bfloat16>(A.out_type, A.head_dim, wide);
  const int64_t blocks = std::min<int64_t>((a.items + THREADS / 32 - 1) / (THREADS / 32), 2 * (int64_t)ctx->sm_count);  // (what is resident)
  return launch(ctx, kern, dim3((unsigned)blocks), THREADS, 0, 1, a);
}
