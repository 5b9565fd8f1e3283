// dc_evict.cu -- a cache without the tokens of least accumulated weight.
//
// For a sequence and key/value head of n tokens: all of them when n <= budget;
// otherwise the last `recent` and, of the `old` ones before them, the `need` =
// budget - recent of largest weight (equal ones: lower index), in their order.
//
// k_evict_select: one cluster of blocks does a (sequence, head); each block
// holds a slice of the old weights, mapped to whole numbers of the same order,
// in shared memory.  The need-th largest is found digit by digit (four digits
// of eight bits, most significant first): the blocks count their slices'
// digits, add the counts to each other's totals through distributed shared
// memory, and all choose the same digit.  Then each block knows how many kept tokens lie before
// its slice and places its own.  Weights are read once.  Counting goes to eight
// copies of the counters, since most weights share their leading bits and
// would otherwise queue for one.  What bounds it is latency: barriers, and the
// first fetch of each instruction, which is why its loops are not unrolled.
// A thread reads four neighbouring weights at once: a call on 8 heads of 131072
// tokens, 16 blocks each, takes 56 us, about 28 of them here, and took 59 with one
// at a time (and then 73 with 8 blocks each, 71 with 1024 threads a block, 74 with 32
// copies).
//
// k_evict_copy: the kept rows, in blocks of about 32 KB of keys and values, all
// of a block's loads in flight together.  Bound by HBM: only kept rows are
// read and written.  Blocks of the heads of one run of places are neighbours,
// since their rows lie side by side.  (16 x 8 heads of 8192 kept rows of 256 bytes:
// 196 us, 5.6 TB/s.)
#include <algorithm>

#include "dc_cache.cuh"

namespace {

using namespace dcc;

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int DIGITS = 256;
constexpr int MAX_CLUSTER = 16;
constexpr int COPIERS = 256;  // threads of a copying block
constexpr int EACH = 4;       // 16-byte pieces of keys and of values that each holds
constexpr int SLICE = 16384;  // weights of a block kept on chip; those of a longer slice are read each time
constexpr int COPIES = 8;     // of the counters

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
  int kv_heads, cache, budget, recent, cluster, slice;
  int pieces, rows, runs;  // 16-byte pieces of a row, rows of a copying block, its blocks a head
  uint32_t inverse;        // ceil(2^32 / pieces)
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
// Adds v to the int at shared address p of block `rank`.
__device__ __forceinline__ void peer_add(const int* p, uint32_t rank, int v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(dcp::smem_u32(p)), "r"(rank));
  asm volatile("red.relaxed.cluster.shared::cluster.add.s32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
// Whole numbers in the order of the floats: NaN below -inf, -0 equal to 0.
__device__ __forceinline__ uint32_t ordered(float f) {
  uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0;
  if (u == 0x80000000u) u = 0;
  return u >> 31 ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(THREADS) k_evict_select(const __grid_constant__ EvArgs a) {
  extern __shared__ __align__(16) uint32_t slice[];  // the block's weights
  __shared__ __align__(16) int counters[COPIES * DIGITS];
  __shared__ __align__(16) int totals[4][DIGITS];  // the cluster's counts of each pass
  __shared__ int warp_gt[WARPS], warp_eq[WARPS];
  __shared__ int block_n[2];        // the slice's weights above and equal to the last one kept
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

  // (whole clusters take one way: n is their sequence's)
  if (n <= a.budget) {
    for (int i = rank * THREADS + tid; i < n; i += a.cluster * THREADS) {
      index[i] = i;
      acc_out[i] = acc[i];
    }
    return;
  }
  const int old = n - a.recent, need = a.budget - a.recent;  // recent <= budget < n
  for (int i = rank * THREADS + tid; i < a.recent; i += a.cluster * THREADS) {
    index[need + i] = old + i;
    acc_out[need + i] = acc[old + i];
  }
  if (need == 0) return;
  const int lo = min(old, (int)rank * a.slice), size = min(old, lo + a.slice) - lo;
  const bool on_chip = a.slice <= SLICE;
  if (tid < DIGITS) reinterpret_cast<int4*>(totals)[tid] = make_int4(0, 0, 0, 0);
  if (a.cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (waited for below)
  if (on_chip) {
#pragma unroll 1
    for (int i0 = tid; i0 < size; i0 += 4 * THREADS) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; j++) x[j] = i0 + j * THREADS < size ? acc[lo + i0 + j * THREADS] : 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (i0 + j * THREADS < size) slice[i0 + j * THREADS] = ordered(x[j]);
    }
  }
  auto weight = [&](int i) { return on_chip ? slice[i] : ordered(__ldg(acc + lo + i)); };
  // Four neighbours from i (a multiple of four) up to `end`, behind which they hold anything.
  auto four = [&](int i, int end, uint32_t (&u)[4]) {
    if (on_chip) {
      const uint4 x = *reinterpret_cast<const uint4*>(slice + i);
      u[0] = x.x, u[1] = x.y, u[2] = x.z, u[3] = x.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) u[j] = i + j < end ? ordered(__ldg(acc + lo + i + j)) : 0;
    }
  };
  uint32_t top = 0;  // the digits found
  int left = need;   // to be taken of the weights that share them
#pragma unroll 1
  for (int pass = 0; pass < 4; pass++) {
    const int shift = 24 - 8 * pass;
    reinterpret_cast<int4*>(counters)[tid] = make_int4(0, 0, 0, 0);
    __syncthreads();
    int* mine = counters + (lane & (COPIES - 1)) * DIGITS;
#pragma unroll 1
    for (int i0 = 4 * tid; i0 < size; i0 += 4 * THREADS) {
      uint32_t u[4];
      four(i0, size, u);
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (i0 + j < size && (pass == 0 || (u[j] >> (shift + 8)) == top))
          atomicAdd(mine + ((u[j] >> shift) & 255), 1);
    }
    __syncthreads();
    int* total = totals[pass];
    if (a.cluster > 1 && pass == 0) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid < DIGITS) {
      int c = 0;
#pragma unroll
      for (int j = 0; j < COPIES; j++) c += counters[j * DIGITS + tid];
      // (a few digits hold all the weights: most lanes have nothing to add)
      if (a.cluster == 1)
        total[tid] = c;
      else if (c)
        for (int r = 0; r < a.cluster; r++) peer_add(&total[tid], (rank + r) & (a.cluster - 1), c);
    }
    if (a.cluster > 1)
      cluster_sync();
    else
      __syncthreads();
    // every warp finds the digit: lane's are 255 - 8 lane and the seven below,
    // the largest first
    int sum = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) sum += total[255 - 8 * lane - j];
    int before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(~0u, before, o);
      if (lane >= o) before += x;
    }
    before -= sum;
    const int owner = __ffs(__ballot_sync(~0u, before < left && before + sum >= left)) - 1;
    left -= __shfl_sync(~0u, before, owner);
    // of the owner's eight digits (lanes 0 to 7 look at one each)
    const int c8 = lane < 8 ? total[255 - 8 * owner - lane] : 0;
    int upto = c8;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      const int x = __shfl_up_sync(~0u, upto, o);
      if (lane >= o) upto += x;
    }
    const int at = __ffs(__ballot_sync(~0u, lane < 8 && upto >= left)) - 1;
    left -= __shfl_sync(~0u, upto - c8, at);
    top = top << 8 | (255 - 8 * owner - at);
  }
  // every kept weight is above `top`, or one of the first `left` equal to it.
  // A warp takes a run of the slice; counts of both before it:
  const int run = (size + WARPS * 32 - 1) / (WARPS * 32) * 32;
  const int r0 = min(size, warp * run), r1 = min(size, r0 + run);
  int gt = 0, eq = 0;
#pragma unroll 1
  for (int i = r0 + 4 * lane; i < r1; i += 128) {
    uint32_t u[4];
    four(i, r1, u);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      gt += i + j < r1 && u[j] > top;
      eq += i + j < r1 && u[j] == top;
    }
  }
  gt = __reduce_add_sync(~0u, gt), eq = __reduce_add_sync(~0u, eq);
  if (lane == 0) warp_gt[warp] = gt, warp_eq[warp] = eq;
  __syncthreads();
  const int wg = lane < WARPS ? warp_gt[lane] : 0, we = lane < WARPS ? warp_eq[lane] : 0;
  int g = __reduce_add_sync(~0u, lane < warp ? wg : 0), e = __reduce_add_sync(~0u, lane < warp ? we : 0);
  if (a.cluster > 1) {
    if (warp == 0) {
      const int x = __reduce_add_sync(~0u, wg), y = __reduce_add_sync(~0u, we);
      if (lane == 0) block_n[0] = x, block_n[1] = y;
    }
    cluster_sync();
    const bool peer = lane < (int)rank;
    g += __reduce_add_sync(~0u, peer ? peer_int(&block_n[0], lane) : 0);
    e += __reduce_add_sync(~0u, peer ? peer_int(&block_n[1], lane) : 0);
    // (no block ends before the others have read its counts: waited for below)
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  const unsigned below = (1u << lane) - 1;
#pragma unroll 2
  for (int i = r0 + lane; i - lane < r1; i += 32) {
    const bool in = i < r1;
    const uint32_t u = in ? weight(i) : 0;
    const unsigned mg = __ballot_sync(~0u, in && u > top), me = __ballot_sync(~0u, in && u == top);
    const int eb = e + __popc(me & below);
    if (in && (u > top || (u == top && eb < left))) {
      const int at = g + __popc(mg & below) + min(eb, left);
      index[at] = lo + i;
      acc_out[at] = __ldg(acc + lo + i);
    }
    g += __popc(mg);
    e += __popc(me);
  }
  if (a.cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__global__ void __launch_bounds__(COPIERS, 4) k_evict_copy(const __grid_constant__ EvArgs a) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int id = blockIdx.x;
  const int h = id % a.kv_heads;
  id /= a.kv_heads;
  const int run = id % a.runs, b = id / a.runs;
  const int kept = min(max(0, min(a.lens[b], a.cache)), a.budget);
  const int i0 = run * a.rows, pieces = min(a.rows, kept - i0) * a.pieces;
  if (pieces <= 0) return;
  const int32_t* index = a.index + b * a.idx_seq + h * a.idx_head + i0;
  const uint8_t *k = a.k + b * a.k_seq + h * a.k_head, *v = a.v + b * a.v_seq + h * a.v_head;
  uint8_t *ko = a.k_out + b * a.ko_seq + h * a.ko_head, *vo = a.v_out + b * a.vo_seq + h * a.vo_head;
  uint4 x[EACH], y[EACH];
  int row[EACH], off[EACH];
  int64_t token[EACH];
#pragma unroll
  for (int j = 0; j < EACH; j++) {
    const int p = j * COPIERS + threadIdx.x;
    row[j] = a.pieces == 1 ? p : __umulhi(p, a.inverse);  // p / pieces: exact for p < 2^16
    off[j] = (p - row[j] * a.pieces) * 16;
    token[j] = p < pieces ? index[row[j]] : -1;
  }
#pragma unroll
  for (int j = 0; j < EACH; j++)
    if (token[j] >= 0) {
      x[j] = *reinterpret_cast<const uint4*>(k + token[j] * a.k_tok + off[j]);
      y[j] = *reinterpret_cast<const uint4*>(v + token[j] * a.v_tok + off[j]);
    }
#pragma unroll
  for (int j = 0; j < EACH; j++)
    if (token[j] >= 0) {
      *reinterpret_cast<uint4*>(ko + (int64_t)(i0 + row[j]) * a.ko_tok + off[j]) = x[j];
      *reinterpret_cast<uint4*>(vo + (int64_t)(i0 + row[j]) * a.vo_tok + off[j]) = y[j];
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
  if ((es != 2 && es != 4) || A.head_dim < 1 || (int64_t)A.head_dim * es % 16 || A.head_dim > COPIERS * EACH * 16 / es)
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
  const std::initializer_list<Dim> dk = {
      {A.batch, A.ko_seq}, {most, A.ko_tok}, {A.kv_heads, A.ko_head}, {A.head_dim, 1}};
  const std::initializer_list<Dim> dv = {
      {A.batch, A.vo_seq}, {most, A.vo_tok}, {A.kv_heads, A.vo_head}, {A.head_dim, 1}};
  const std::initializer_list<Dim> da = {{A.batch, A.acco_seq}, {A.kv_heads, A.acco_head}, {most, 1}};
  const std::initializer_list<Dim> di = {{A.batch, A.idx_seq}, {A.kv_heads, A.idx_head}, {most, 1}};
  const Span out[5] = {span(A.k_out, es, dk), span(A.v_out, es, dv), span(A.acc_out, 4, da), span(A.index, 4, di),
                       span(A.lens_out, 4, {{A.batch, 1}})};
  for (const Span& o : out) {
    for (const Span& i : in)
      if (!o.ok || !i.ok || o.meets(i))
        return dc_fail(ctx, DC_E_INVAL, "cache_evict: a negative stride, or an output overlaps an input");
    // (k_out and v_out may be interleaved in one buffer)
    for (const Span& q : out)
      if (&q < &o && !(&o == &out[1] && &q == &out[0] ? twins_apart(q, o, es, dk, dv) : !o.meets(q)))
        return dc_fail(ctx, DC_E_INVAL, "cache_evict: two outputs overlap");
  }
  if (!apart(dk) || !apart(dv) || !apart(da) || !apart(di))
    return dc_fail(ctx, DC_E_INVAL, "cache_evict: two elements of an output share an address");
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
  a.kv_heads = A.kv_heads, a.cache = A.cache, a.budget = A.budget, a.recent = A.recent;
  a.pieces = A.head_dim * es / 16;
  a.inverse = (uint32_t)(((1ull << 32) + a.pieces - 1) / a.pieces);
  a.rows = COPIERS * EACH / a.pieces;
  a.runs = (most + a.rows - 1) / a.rows;
  // blocks of a head: one for each 4096 tokens while the call does not fill
  // every SM (16 sequences x 8 heads of 16384 tokens: 35 us in clusters of two,
  // 41 in fours, 63 in eights), and enough to hold the weights on chip
  const int64_t heads = (int64_t)A.batch * A.kv_heads;
  int cl = 1;
  while (cl < MAX_CLUSTER && ((heads * cl < ctx->sm_count && A.cache > 4096 * cl) || A.cache > SLICE * cl)) cl <<= 1;
  a.cluster = cl;
  a.slice = (std::max(1, A.cache) + cl - 1) / cl;
  if (heads * std::max(a.runs, cl) > INT32_MAX) return dc_fail(ctx, DC_E_INVAL, "cache_evict: too many blocks");
  if (cl > 8)
    DC_CUDA(ctx, cudaFuncSetAttribute((const void*)k_evict_select, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  if (int rc = launch(ctx, k_evict_select, dim3((unsigned)(heads * cl)), THREADS, a.slice <= SLICE ? (a.slice + 3) / 4 * 16 : 0, cl, a))
    return rc;
  return most ? launch(ctx, k_evict_copy, dim3((unsigned)(heads * a.runs)), COPIERS, 0, 1, a) : DC_OK;
}
