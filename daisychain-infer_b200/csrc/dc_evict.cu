// dc_evict.cu -- a cache without the tokens of least accumulated weight.
//
// For a sequence and key/value head of n tokens: all of them when n <= budget;
// otherwise the last `recent` and, of the `old` ones before them, the `need` =
// budget - recent of largest weight (equal ones: lower index), in their order.
//
// One cluster of blocks does a (sequence, head): each block holds a slice of the
// old weights, mapped to whole numbers of the same order, in shared memory.
// The need-th largest is found digit by digit (four digits of eight bits, most
// significant first): the blocks count their slices' digits, read each other's
// counts through distributed shared memory, and all choose the same digit.  Then
// each block knows how many kept tokens lie before its slice, places its own,
// and the cluster copies the kept rows, each block an even share.  So weights
// are read once, only kept rows are read and written, and it is one launch.
//
// Bound by HBM through the kept rows' copies (16-byte pieces, eight in flight a
// thread); the selection costs a few microseconds.  Counting is by lane: a
// digit has one counter for each of the 32 lanes, in its own bank, since most
// weights share their leading bits and would otherwise queue for one counter.
#include <algorithm>

#include "dc_cache.cuh"

namespace {

using namespace dcc;

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int DIGITS = 256;
constexpr int MAX_CLUSTER = 16;
constexpr int SLICE = 32768;  // weights of a block kept on chip; a longer slice is read from memory each time

struct EvArgs {
  const uint8_t *k, *v;
  const float* acc;
  const int32_t* lens;
  uint8_t *k_out, *v_out;
  float* acc_out;
  int32_t *index, *lens_out;
  // (strides of k and v in bytes)
  int64_t k_seq, k_tok, k_head, v_seq, v_tok, v_head, acc_seq, acc_head;
  int64_t ko_seq, ko_tok, ko_head, vo_seq, vo_tok, vo_head, acco_seq, acco_head, idx_seq, idx_head;
  int kv_heads, pieces, cache, budget, recent, cluster, slice;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The int at shared address p of block `rank` of the cluster.
__device__ __forceinline__ int peer_int(const int* p, uint32_t rank) {
  uint32_t at;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(dcp::smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
// Whole numbers in the order of the floats: NaN below -inf, -0 equal to 0.
__device__ __forceinline__ uint32_t ordered(float f) {
  uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
  if (u == 0x80000000u) u = 0;
  return u >> 31 ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(THREADS) k_cache_evict(const __grid_constant__ EvArgs a) {
  extern __shared__ uint32_t keys[];         // the slice's weights as whole numbers
  __shared__ int lanes[DIGITS * 32];         // counts by digit and lane
  __shared__ int count[4][DIGITS];           // the block's counts of each pass, for the cluster
  __shared__ int chosen[2];                  // a pass's digit, and what is still to be taken of it
  __shared__ int warp_gt[WARPS + 1], warp_eq[WARPS + 1];
  __shared__ int block_n[2];                 // the slice's weights above and equal to the last one kept
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int bh = blockIdx.x / a.cluster, b = bh / a.kv_heads, h = bh - b * a.kv_heads;
  const int n = max(0, min(a.lens[b], a.cache)), kept = min(n, a.budget);
  const float* acc = a.acc + b * a.acc_seq + h * a.acc_head;
  float* acc_out = a.acc_out + b * a.acco_seq + h * a.acco_head;
  int32_t* index = a.index + b * a.idx_seq + h * a.idx_head;
  if (h == 0 && rank == 0 && tid == 0) a.lens_out[b] = kept;

  if (n <= a.budget) {  // (the whole cluster: n is its sequence's)
    for (int i = rank * THREADS + tid; i < n; i += a.cluster * THREADS) {
      index[i] = i;
      acc_out[i] = acc[i];
    }
  } else {
    const int old = n - a.recent, need = a.budget - a.recent;  // recent <= budget < n
    const int lo = min(old, (int)rank * a.slice), size = min(old, lo + a.slice) - lo;
    const bool on_chip = a.slice <= SLICE;
    if (on_chip && need > 0) {
      for (int i = tid; i < size; i += THREADS) keys[i] = ordered(acc[lo + i]);
    }
    auto key = [&](int i) { return on_chip ? keys[i] : ordered(acc[lo + i]); };
    uint32_t top = 0;  // the digits found
    int left = need;   // to be taken of the weights that share them
    if (need > 0) {
#pragma unroll 1
      for (int pass = 0; pass < 4; pass++) {
        const int shift = 24 - 8 * pass;
        for (int i = tid; i < DIGITS * 32; i += THREADS) lanes[i] = 0;
        __syncthreads();
        for (int i = tid; i < size; i += THREADS) {
          const uint32_t u = key(i);
          if (pass == 0 || (u >> (shift + 8)) == top) atomicAdd(&lanes[((u >> shift) & 255) * 32 + lane], 1);
        }
        __syncthreads();
        for (int d = warp; d < DIGITS; d += WARPS) {
          const int c = __reduce_add_sync(~0u, lanes[d * 32 + lane]);
          if (lane == 0) count[pass][d] = c;
        }
        cluster_sync();
        if (warp == 0) {
          // lane's digits are 255 - 8 lane and the seven below, the largest first
          int c[8], s = 0;
#pragma unroll
          for (int j = 0; j < 8; j++) c[j] = 0;
          for (int r = 0; r < a.cluster; r++) {
#pragma unroll
            for (int j = 0; j < 8; j++) c[j] += peer_int(&count[pass][255 - 8 * lane - j], r);
          }
#pragma unroll
          for (int j = 0; j < 8; j++) s += c[j];
          int before = s;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(~0u, before, o);
            if (lane >= o) before += x;
          }
          before -= s;
          if (before < left && before + s >= left) {
            int want = left - before, d = 255 - 8 * lane;
#pragma unroll
            for (int j = 0; j < 7; j++)
              if (255 - 8 * lane - j == d && want > c[j]) {
                want -= c[j];
                d--;
              }
            chosen[0] = d;
            chosen[1] = want;
          }
        }
        __syncthreads();
        top = top << 8 | chosen[0];
        left = chosen[1];
      }
    }
    // every kept weight is above `top`, or one of the first `left` equal to it
    // (need = 0: none).  A warp takes a run of the slice; counts before it:
    const int run = (size + WARPS * 32 - 1) / (WARPS * 32) * 32;
    const int r0 = min(size, warp * run), r1 = min(size, r0 + run);
    if (need > 0) {
      int gt = 0, eq = 0;
      for (int i = r0; i < r1; i += 32) {
        const bool in = i + lane < r1;
        const uint32_t u = in ? key(i + lane) : 0;
        gt += __popc(__ballot_sync(~0u, in && u > top));
        eq += __popc(__ballot_sync(~0u, in && u == top));
      }
      if (lane == 0) warp_gt[warp] = gt, warp_eq[warp] = eq;
      __syncthreads();
      if (tid == 0) {
        int g = 0, e = 0;
        for (int w = 0; w < WARPS; w++) {
          const int x = warp_gt[w], y = warp_eq[w];
          warp_gt[w] = g, warp_eq[w] = e;
          g += x, e += y;
        }
        block_n[0] = g, block_n[1] = e;
      }
      cluster_sync();
      int g = warp_gt[warp], e = warp_eq[warp];
      for (int r = 0; r < (int)rank; r++) g += peer_int(&block_n[0], r), e += peer_int(&block_n[1], r);
      const unsigned below = (1u << lane) - 1;
      for (int i = r0; i < r1; i += 32) {
        const bool in = i + lane < r1;
        const uint32_t u = in ? key(i + lane) : 0;
        const unsigned mg = __ballot_sync(~0u, in && u > top), me = __ballot_sync(~0u, in && u == top);
        const int eb = e + __popc(me & below);
        if (in && (u > top || (u == top && eb < left))) {
          const int at = g + __popc(mg & below) + min(eb, left), token = lo + i + lane;
          index[at] = token;
          acc_out[at] = acc[token];
        }
        g += __popc(mg);
        e += __popc(me);
      }
    }
    for (int i = rank * THREADS + tid; i < a.recent; i += a.cluster * THREADS) {
      index[need + i] = old + i;
      acc_out[need + i] = acc[old + i];
    }
  }
  cluster_sync();  // the index is complete, and no block reads another's counts any more

  // the kept rows: a thread copies one 16-byte piece of a key and of a value row
  // at a time, four rows in flight
  const int per = THREADS / a.pieces;  // rows of a step
  const int r = tid / a.pieces;
  const int64_t piece = (int64_t)(tid - r * a.pieces) * 16;
  if (r >= per) return;
  const uint8_t* k = a.k + b * a.k_seq + h * a.k_head + piece;
  const uint8_t* v = a.v + b * a.v_seq + h * a.v_head + piece;
  uint8_t* ko = a.k_out + b * a.ko_seq + h * a.ko_head + piece;
  uint8_t* vo = a.v_out + b * a.vo_seq + h * a.vo_head + piece;
  const int step = per * a.cluster;
  for (int i0 = rank * per + r; i0 < kept; i0 += 4 * step) {
    uint4 x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int i = i0 + j * step;
      if (i < kept) {
        const int64_t token = __ldcg(index + i);
        x[j] = *reinterpret_cast<const uint4*>(k + token * a.k_tok);
        y[j] = *reinterpret_cast<const uint4*>(v + token * a.v_tok);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t i = i0 + j * step;
      if (i < kept) {
        *reinterpret_cast<uint4*>(ko + i * a.ko_tok) = x[j];
        *reinterpret_cast<uint4*>(vo + i * a.vo_tok) = y[j];
      }
    }
  }
}

}  // namespace

extern "C" int dc_cache_evict_dev(dc_ctx* ctx, const dc_cache_evict* p) {
  if (!ctx || !p) return dc_fail(ctx, DC_E_INVAL, "cache_evict: bad arguments");
  const dc_cache_evict& A = *p;
  if (A.batch < 0 || A.kv_heads < 1 || (int64_t)A.batch * A.kv_heads > (1 << 20) || A.cache < 0 || A.cache > (1 << 30))
    return dc_fail(ctx, DC_E_INVAL, "cache_evict: batch %d, kv_heads %d, cache %d", A.batch, A.kv_heads, A.cache);
  if (A.budget < 0 || A.recent < 0 || A.recent > A.budget)
    return dc_fail(ctx, DC_E_INVAL, "cache_evict: recent %d, budget %d", A.recent, A.budget);
  const int es = A.elem_bytes;
  if ((es != 2 && es != 4) || A.head_dim < 1 || (int64_t)A.head_dim * es % 16 || A.head_dim > THREADS * 16 / es)
    return dc_fail(ctx, DC_E_INVAL, "cache_evict: rows of %d elements of %d bytes", A.head_dim, es);
  if (!A.batch) return DC_OK;
  const int most = std::min(A.budget, A.cache);  // tokens that may be written
  if (!A.lens || !A.lens_out || (most && (!A.k || !A.v || !A.acc || !A.k_out || !A.v_out || !A.acc_out || !A.index)))
    return dc_fail(ctx, DC_E_INVAL, "cache_evict: null buffer");
  auto row_ok = [&](const void* p, int64_t seq, int64_t n, int64_t tok, int64_t head) {
    return aligned(p, es, 16, {{A.batch, seq}, {n, tok}, {A.kv_heads, head}});
  };
  if (most && (!row_ok(A.k, A.k_seq, A.cache, A.k_tok, A.k_head) || !row_ok(A.v, A.v_seq, A.cache, A.v_tok, A.v_head) ||
               !row_ok(A.k_out, A.ko_seq, most, A.ko_tok, A.ko_head) ||
               !row_ok(A.v_out, A.vo_seq, most, A.vo_tok, A.vo_head)))
    return dc_fail(ctx, DC_E_INVAL, "cache_evict: k and v rows must begin on 16-byte boundaries");
  const Span in[4] = {
      span(A.k, es, {{A.batch, A.k_seq}, {A.cache, A.k_tok}, {A.kv_heads, A.k_head}, {A.head_dim, 1}}),
      span(A.v, es, {{A.batch, A.v_seq}, {A.cache, A.v_tok}, {A.kv_heads, A.v_head}, {A.head_dim, 1}}),
      span(A.acc, 4, {{A.batch, A.acc_seq}, {A.kv_heads, A.acc_head}, {A.cache, 1}}), span(A.lens, 4, {{A.batch, 1}})};
  const Span out[5] = {
      span(A.k_out, es, {{A.batch, A.ko_seq}, {most, A.ko_tok}, {A.kv_heads, A.ko_head}, {A.head_dim, 1}}),
      span(A.v_out, es, {{A.batch, A.vo_seq}, {most, A.vo_tok}, {A.kv_heads, A.vo_head}, {A.head_dim, 1}}),
      span(A.acc_out, 4, {{A.batch, A.acco_seq}, {A.kv_heads, A.acco_head}, {most, 1}}),
      span(A.index, 4, {{A.batch, A.idx_seq}, {A.kv_heads, A.idx_head}, {most, 1}}), span(A.lens_out, 4, {{A.batch, 1}})};
  for (const Span& o : out) {
    for (const Span& i : in)
      if (!o.ok || !i.ok || o.meets(i))
        return dc_fail(ctx, DC_E_INVAL, "cache_evict: a negative stride, or an output overlaps an input");
    // (k_out and v_out may be interleaved in one buffer, so only the same address is refused there)
    for (const Span& q : out)
      if (&q < &o && o.meets(q) && !(&o == &out[1] && &q == &out[0] && o.lo != q.lo))
        return dc_fail(ctx, DC_E_INVAL, "cache_evict: two outputs overlap");
  }
  DeviceGuard guard;
  if (int rc = guard.enter(ctx)) return rc;

  EvArgs a;
  a.k = (const uint8_t*)A.k, a.v = (const uint8_t*)A.v, a.acc = A.acc, a.lens = A.lens;
  a.k_out = (uint8_t*)A.k_out, a.v_out = (uint8_t*)A.v_out, a.acc_out = A.acc_out;
  a.index = A.index, a.lens_out = A.lens_out;
  a.k_seq = A.k_seq * es, a.k_tok = A.k_tok * es, a.k_head = A.k_head * es;
  a.v_seq = A.v_seq * es, a.v_tok = A.v_tok * es, a.v_head = A.v_head * es;
  a.ko_seq = A.ko_seq * es, a.ko_tok = A.ko_tok * es, a.ko_head = A.ko_head * es;
  a.vo_seq = A.vo_seq * es, a.vo_tok = A.vo_tok * es, a.vo_head = A.vo_head * es;
  a.acc_seq = A.acc_seq, a.acc_head = A.acc_head, a.acco_seq = A.acco_seq, a.acco_head = A.acco_head;
  a.idx_seq = A.idx_seq, a.idx_head = A.idx_head;
  a.kv_heads = A.kv_heads, a.pieces = A.head_dim * es / 16, a.cache = A.cache;
  a.budget = A.budget, a.recent = A.recent;
  // blocks of a head: until the call fills every SM, but no fewer than 128
  // tokens a block
  const int64_t heads = (int64_t)A.batch * A.kv_heads;
  int cl = 1;
  while (cl < MAX_CLUSTER && heads * cl < ctx->sm_count && A.cache >= 256 * cl) cl <<= 1;
  a.cluster = cl;
  a.slice = (std::max(1, A.cache) + cl - 1) / cl;
  if (cl > 8)
    DC_CUDA(ctx, cudaFuncSetAttribute((const void*)k_cache_evict, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  const int smem = a.slice <= SLICE ? a.slice * 4 : 0;
  return launch(ctx, k_cache_evict, dim3((unsigned)(heads * cl)), THREADS, smem, cl, a);
}
