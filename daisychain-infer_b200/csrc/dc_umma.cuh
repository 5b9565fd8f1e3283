// dc_umma.cuh -- 16-bit tcgen05 products, TMEM access and tensor maps (sm_100a).
//
// Shared by the attention over a batch's cache (dc_prefix.cu) and the
// accumulation of attention weights (dc_weights.cu).  Operands are 64-element
// (128-byte) wide panels with the 128-byte swizzle, accumulators f32 in TMEM.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include "dc_internal.cuh"
#include "dc_ptx.cuh"

namespace dcu {

constexpr int PANEL = 64;  // elements of one panel row: 128 bytes, one swizzle row

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dcp::smem_u32(dst)),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(dcp::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dcp::smem_u32(dst)),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(dcp::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, int v,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];" ::"r"(dcp::smem_u32(dst)),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(dcp::smem_u32(bar))
      : "memory");
}

// Shared-memory descriptor of a 128B-swizzled operand whose 8-row groups lie
// 1024 bytes apart.  K-major (rows are the M or N index, 64 K elements a row):
// `lead` is unused.  MN-major (rows are the K index, 64 M or N elements a
// row): `lead` is the distance in bytes to the next 64 elements.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lead) {
  uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lead >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version (sm_100)
  d |= (uint64_t)2 << 61;  // SWIZZLE_128B
  return d;
}
// Instruction descriptor of kind::f16: f32 accumulators, A and B both bf16 or
// both f16, A K-major, B K-major or (b_mn) MN-major, M = 128.
__device__ __forceinline__ constexpr uint32_t idesc(bool bf16, int n, bool b_mn) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((128u >> 4) << 24);
}
// True in one lane of a converged warp, for `if (elect())` around products and
// commits: the compiler knows this form, and their operands stay in uniform
// registers (eight products issue in 100 to 165 cycles; under `if (lane == 0)` in
// 385, which then bounded the softmax kernels).
__device__ __forceinline__ bool elect() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e != 0;
}
// A value that is the same in all lanes, as one the compiler knows to be.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(~0u, v, 0); }
// A wait of a whole warp: true where every lane's wait was met.  A plain test goes
// first: where the barrier is met it takes 41 cycles, the suspending one 89.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status) {
  uint32_t met;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(met)
      : "r"(dcp::smem_u32(bar)), "r"(parity)
      : "memory");
  return __all_sync(~0u, met) || __all_sync(~0u, dcp::mbar_wait(bar, parity, status));
}
// The same where the lanes wait for different barriers, and all go on to use what any
// of them guards: a vote orders no memory between lanes, __syncwarp does.
__device__ __forceinline__ bool warp_wait_each(uint64_t* bar, uint32_t parity, int* status) {
  const bool met = warp_wait(bar, parity, status);
  __syncwarp();
  return met;
}
// D (TMEM) (+)= A (shared) x B (shared)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
// D (TMEM) (+)= A (TMEM) x B (shared)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
// One arrival on `bar` once the products that this lane issued so far are complete.
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   dcp::smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dcp::smem_u32(slot)),
               "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

#define DCU_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define DCU_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 32 consecutive f32 columns of this thread's TMEM lane (the warp's quarter is
// in `addr`); asynchronous until wait_ld.
__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : DCU_R8(r, 0), DCU_R8(r, 8), DCU_R8(r, 16), DCU_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::DCU_I8(r, 0),
      DCU_I8(r, 8), DCU_I8(r, 16), DCU_I8(r, 24), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : DCU_R8(r, 0), DCU_R8(r, 8)
      : "r"(addr));
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::DCU_I8(
          r, 0),
      DCU_I8(r, 8), "r"(addr)
      : "memory");
}
// The loads' registers pass through the wait, so that no use of them can be
// scheduled before it.
template <int N>
__device__ __forceinline__ void wait_ld(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two f32 in a register pair, and the packed operations on them.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x of both halves on the multiply-add pipe, for where the exponential unit
// (16 a cycle and SM) is what a kernel waits for: x = n + f with n whole and |f|
// <= 1/2 (n by adding 1.5 x 2^23), 2^f by its best polynomial of degree five (7.5e-8
// relative, from a Remez iteration; 2.1e-7 with the f32 roundings, as the unit's
// own 2.4e-7), 2^n from its exponent field.  0 from x = -126.5 down, inf from 127.5
// up, NaN for NaN.
__device__ __forceinline__ F2 ex2_fma(F2 x) {
  float2 v = split(x);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(-127.0f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(-127.0f));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v.x) : "f"(128.0f));
  asm("min.NaN.f32 %0, %0, %1;" : "+f"(v.y) : "f"(128.0f));
  const F2 y = f2(v.x, v.y), t = add2(y, f2(12582912.0f, 12582912.0f));
  const F2 f = fma2(add2(t, f2(-12582912.0f, -12582912.0f)), f2(-1.0f, -1.0f), y);
  F2 p = fma2(f, f2(0.0013276472454890609f, 0.0013276472454890609f), f2(0.009675540961325169f, 0.009675540961325169f));
  p = fma2(p, f, f2(0.05550713092088699f, 0.05550713092088699f));
  p = fma2(p, f, f2(0.24022120237350464f, 0.24022120237350464f));
  p = fma2(p, f, f2(0.6931469440460205f, 0.6931469440460205f));
  p = fma2(p, f, f2(1.0000001192092896f, 1.0000001192092896f));
  const float2 w = split(t);
  return mul2(p, f2(__int_as_float((__float_as_int(w.x) << 23) + 0x3f800000),
                    __int_as_float((__float_as_int(w.y) << 23) + 0x3f800000)));
}

// A tensor map over `rank` dimensions of a 16-bit tensor; strides[i] (bytes)
// is that of dims[i + 1].  A dimension of one element may have any stride, so
// the map is given a harmless one.  False when the driver refuses the map.
static inline bool encode(CUtensorMap* map, const void* base, bool bf16, int rank, const uint64_t* dims,
                          const uint64_t* strides, const uint32_t* box) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess) p = nullptr;
    return (PFN_cuTensorMapEncodeTiled_v12000)p;
  }();
  if (!fn) return false;
  cuuint64_t d[5], s[4];
  cuuint32_t b[5], es[5];
  for (int i = 0; i < rank; i++) {
    d[i] = dims[i];
    b[i] = box[i];
    es[i] = 1;
    if (i) s[i - 1] = dims[i] == 1 ? 2 * ((dims[0] + 7) / 8 * 8) : strides[i - 1];
  }
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
            const_cast<void*>(base), d, s, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace dcu
