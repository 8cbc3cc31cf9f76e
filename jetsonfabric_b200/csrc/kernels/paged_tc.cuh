// tcgen05 building blocks of the paged attention kernels: shared-memory and
// instruction descriptors, MMA issue, tensor-memory loads and stores, packed
// f32 arithmetic. The MMA and commit wrappers are executed by a converged
// warp, one elected lane issuing.
#pragma once

#include <type_traits>

#include "paged.cuh"

namespace jfb {
namespace paged {

constexpr uint32_t kHalfBytes = kTileKeys * 128;  // one [128 rows][64] half of a tile

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// All of an SM's tensor memory, by one warp.
__device__ __forceinline__ void tmem_alloc(uint32_t * slot) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Matrix descriptors of operands in the 128-byte swizzle (bits 61-63 = 2, bit
// 46 the sm_100 version), 8-row groups 1024 bytes apart. K-major: rows are the
// M or N index, 64 consecutive K values a row; a K step of 16 adds 32 bytes.
// MN-major: rows are the K index, 64 consecutive N values a row, the next 64
// one half (lbo) further; a K step of 16 adds two groups, 2048 bytes.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
    return uint64_t((addr & 0x3FFFF) >> 4) | uint64_t(1) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 | uint64_t(2) << 61;
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr) {
    return uint64_t((addr & 0x3FFFF) >> 4) | uint64_t(kHalfBytes >> 4) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 |
           uint64_t(2) << 61;
}

// kind::f16 with f32 accumulation, A and B both f16 or both bf16, M = 128.
template <typename T>
constexpr uint32_t instr_desc(uint32_t n, bool b_mn_major) {
    const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | (b_mn_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

// D (+)= A B, A and B in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// The same with A in tensor memory: lane = row, each column a pair of K values.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// `bar` completes a phase when every MMA issued before has finished.
__device__ __forceinline__ void mma_commit(uint64_t * bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}

// The 128 x 128 scores of two K-major tiles of D columns.
template <typename T, int D>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t at = (kk >> 2) * kHalfBytes + (kk & 3) * 32;
        mma_ss(d, desc_k_major(a + at), desc_k_major(b + at), instr_desc<T>(kTileKeys, false), kk > 0);
    }
}

#define JFB_R8(r, i) "=f"(r[i]), "=f"(r[i + 1]), "=f"(r[i + 2]), "=f"(r[i + 3]), "=f"(r[i + 4]), "=f"(r[i + 5]), "=f"(r[i + 6]), "=f"(r[i + 7])
#define JFB_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])

// 32 consecutive f32 columns of this thread's lane (valid after tmem_wait_ld).
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float * r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : JFB_R8(r, 0), JFB_R8(r, 8), JFB_R8(r, 16), JFB_R8(r, 24)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float * r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : JFB_R8(r, 0), JFB_R8(r, 8)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t * r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        JFB_W8(r, 0), JFB_W8(r, 8)
        : "memory");
}
#undef JFB_R8
#undef JFB_W8
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two f32 operations in one instruction, each rounded like the scalar one.
__device__ __forceinline__ void fma2(float & d0, float & d1, float a0, float a1, float b, float c) {
    asm("{\n\t.reg .b64 a, b, c;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void fma2(float & d0, float & d1, float a0, float a1, float b, float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %6};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void add2(float & d0, float & d1, float a0, float a1) {
    asm("{\n\t.reg .b64 a, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 d, {%0, %1};\n\t"
        "add.rn.f32x2 d, d, a;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "+f"(d0), "+f"(d1)
        : "f"(a0), "f"(a1));
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Query rows as (head_dim, heads, rows): boxes of 64 elements x the group x
// `tokens` rows, so a box's rows are packed rows (token, head of the group).
inline bool query_map(CUtensorMap & map, const View & v, const void * q, uint64_t q_stride, uint32_t heads, uint32_t tokens) {
    PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[3] = {v.head_dim, heads, v.rows};
    const cuuint64_t strides[2] = {uint64_t(v.head_dim) * 2, q_stride * 2};
    const cuuint32_t box[3] = {64, v.group, tokens};
    const cuuint32_t elem[3] = {1, 1, 1};
    std::memset(&map, 0, sizeof(map));
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(q), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace paged
}  // namespace jfb
