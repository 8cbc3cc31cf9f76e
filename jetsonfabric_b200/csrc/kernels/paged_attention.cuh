// What the paged attention kernels share: parameters, row outputs, workspace
// layout and the checks of row arrays.
#pragma once

#include "paged.cuh"

namespace jfb {
namespace paged {

// Workspace: two arrival counters per CTA (an item split over CTAs counts at
// its first one, in the tcgen05 kernel per row tile), then two slots per CTA for the parts of the items that
// begin before it and that end behind it: [256 rows][128] sums and [256]
// (maximum, sum), f32.
constexpr uint64_t kCounterBytes = 4096;
constexpr uint64_t kSlotFloats = 256 * (128 + 2);

struct AttentionParams {
    View view;
    const void * q;
    void * out;
    float * lse;
    uint64_t q_stride, out_stride;
    uint32_t heads, group, window;
    float scale;
    uint32_t * counters;
    float * partial;
};

// Where packed row r of the walk's item goes.
template <typename T>
struct RowsOut {
    T * out;  // nullptr: no such row
    uint64_t at;
    __device__ __forceinline__ RowsOut(const AttentionParams & p, const Walk & w, uint32_t r) {
        const bool valid = r < w.s.count * p.group;
        const uint32_t row = w.s.q0 + (valid ? r / p.group : 0u), head = w.kv_head * p.group + (valid ? r % p.group : 0u);
        out = valid ? static_cast<T *>(p.out) + uint64_t(row) * p.out_stride + uint64_t(head) * p.view.head_dim : nullptr;
        at = uint64_t(row) * p.heads + head;
    }
    // four columns of sums over the softmax sum; a row that saw nothing is zero
    __device__ __forceinline__ void store4(uint32_t d, float4 a, float sum, uint32_t head_dim) const {
        if (out == nullptr || d >= head_dim) return;
        const float f = sum != 0.0f ? 1.0f / sum : 0.0f;
        *reinterpret_cast<uint2 *>(out + d) = make_uint2(Num<T>::pack(a.x * f, a.y * f), Num<T>::pack(a.z * f, a.w * f));
    }
    // top is the maximum in units of log 2
    __device__ __forceinline__ void store_lse(const AttentionParams & p, float top, float sum) const {
        if (out != nullptr && p.lse != nullptr) p.lse[at] = sum != 0.0f ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
    }
};

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The tcgen05 kernel of paged_attention_tc.cu.
jfb_status launch_attention_tc(bool half, uint32_t head_dim, const CUtensorMap & k, const CUtensorMap & v, const AttentionParams & p,
                               uint32_t sms, cudaStream_t s);

// Query-shaped rows [rows][heads x head_dim] of 16-bit numbers.
inline jfb_status check_rows(const char * what, const void * x, uint64_t stride, uint32_t rows, uint32_t heads,
                             const jfb_paged_cache & c) {
    if (x == nullptr || (reinterpret_cast<uintptr_t>(x) & 15u) != 0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "%s rows must be given, 16-byte aligned", what);
    }
    if (heads == 0 || heads % c.kv_heads != 0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "%s: %u heads over %u kv heads", what, heads, c.kv_heads);
    }
    if (stride % 8 != 0 || stride < uint64_t(heads) * c.head_dim || stride >= (1ull << 40)) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "%s: a row stride of %llu elements does not fit %u heads of %u", what,
                            static_cast<unsigned long long>(stride), heads, c.head_dim);
    }
    if (rows > 0x7fffffffu || uint64_t(rows) * (heads / c.kv_heads) > 0x7fffffffull) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "%s: too many rows", what);
    }
    return status_ok();
}

}  // namespace paged
}  // namespace jfb
