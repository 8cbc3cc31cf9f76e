// What the paged attention kernels share: parameters, row outputs, workspace
// layout and the checks of row arrays.
#pragma once

#include <type_traits>

#include "paged.cuh"

namespace jfb {
namespace paged {

// Workspace: two arrival counters per CTA (an item split over CTAs counts at
// its first one, in the tcgen05 kernel per row tile), then two slots per CTA for the parts of the items that
// begin before it and that end behind it: [256 rows][128] sums and [256]
// (maximum, sum), f32.
constexpr uint64_t kCounterBytes = 4096;
constexpr uint64_t kSlotFloats = 256 * (128 + 2);

// A row's exponentials and sums refer to a number m (log 2) that was its
// maximum less kHeadroom when it was last set; it is set again when the maximum
// has come to exceed it by more than kSlack + kHeadroom. As operands of the
// second product the exponentials are rounded to the cache's type. f16 has
// nothing below 2^-25, where many weak keys beside a strong one would count in
// the softmax sum and not in the result (2^17 keys of 2^-25.2 each are 0.3 % of
// it), so its exponentials start at 2^7: they stay below 2^15 and none above
// 2^-32 of the row's largest is lost. bf16 has the exponents of f32.
constexpr float kSlack = 8.0f;
template <typename T>
constexpr float kHeadroom = std::is_same<T, __half>::value ? 7.0f : 0.0f;

// The scaled maximum, rounded up: no exponential may lie above it, whatever a
// step of f32 at its size.
__device__ __forceinline__ float scaled_top(float score, float scale2) { return __fmul_ru(score, scale2); }

// Whether the reference m of a row whose maximum is `top` has to be set again.
// The difference of close numbers is exact; it is NaN, hence false, where
// nothing was seen yet.
template <typename T>
__device__ __forceinline__ bool outgrown(float top, float m) {
    return top - m > kSlack + kHeadroom<T>;
}

struct AttentionParams {
    View view;
    const void * q;
    void * out;
    float * lse;
    uint64_t q_stride, out_stride;
    uint32_t heads;
    float scale;
    uint32_t * counters;
    float * partial;
};

// Where a result row goes.
template <typename T>
struct RowsOut {
    T * out;  // nullptr: no such row
    uint64_t at;
    __device__ __forceinline__ RowsOut(const AttentionParams & p, bool valid, uint32_t row, uint32_t head) {
        out = valid ? static_cast<T *>(p.out) + uint64_t(row) * p.out_stride + uint64_t(head) * p.view.head_dim : nullptr;
        at = uint64_t(row) * p.heads + head;
    }
    // two columns of sums over the softmax sum; a row that saw nothing is zero
    __device__ __forceinline__ void store2(uint32_t d, float a, float b, float sum, uint32_t head_dim) const {
        if (out == nullptr || d >= head_dim) return;
        const float f = sum != 0.0f ? 1.0f / sum : 0.0f;
        *reinterpret_cast<uint32_t *>(out + d) = Num<T>::pack(a * f, b * f);
    }
    // sixteen columns, as one 32-byte sector where rows are aligned to it
    __device__ __forceinline__ void store16(uint32_t d, const float * a, float sum, uint32_t head_dim, bool sectors) const {
        if (out == nullptr || d >= head_dim) return;
        const float f = sum != 0.0f ? 1.0f / sum : 0.0f;
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = Num<T>::pack(a[2 * i] * f, a[2 * i + 1] * f);
        if (sectors && d + 16 <= head_dim) {
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + d), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                         "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
        } else {
            *reinterpret_cast<uint4 *>(out + d) = make_uint4(w[0], w[1], w[2], w[3]);
            if (d + 8 < head_dim) *reinterpret_cast<uint4 *>(out + d + 8) = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
    // m is what the sum refers to, in units of log 2
    __device__ __forceinline__ void store_lse(const AttentionParams & p, float m, float sum) const {
        if (out != nullptr && p.lse != nullptr) p.lse[at] = sum != 0.0f ? fmaf(m, kLn2, logf(sum)) : -INFINITY;
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

// Which kernel a (valid) call takes: 1 the tcgen05 one, 0 the few-rows one.
// Exported, not part of the interface: the tests make sure of what they cover.
extern "C" int jfb_paged_attention_uses_tiles(uint32_t rows, uint32_t heads, uint32_t window, const jfb_paged_cache * cache,
                                              const jfb_paged_batch * batch);
extern "C" int jfb_paged_attention_mass_uses_tiles(uint32_t rows, uint32_t heads, const jfb_paged_cache * cache,
                                                   const jfb_paged_batch * batch, uint64_t mass_stride);

// The tcgen05 kernel of paged_attention_tc.cu.
jfb_status launch_attention_tc(const jfb_paged_cache & cache, const CUtensorMap & k, const CUtensorMap & v, AttentionParams p,
                               const Device & device, cudaStream_t s);

// Whether rows of `width` 16-bit elements at two strides share bytes: in an
// address range that both lie in, slices of wider rows of one stride need not.
inline bool rows_overlap(const void * a, uint64_t a_stride, const void * b, uint64_t b_stride, uint32_t rows, uint64_t width) {
    if (rows == 0) return false;
    const uint64_t x = reinterpret_cast<uintptr_t>(a) / 2, y = reinterpret_cast<uintptr_t>(b) / 2;
    if (x + (rows - 1) * a_stride + width <= y || y + (rows - 1) * b_stride + width <= x) return false;
    if (a_stride != b_stride) return true;
    const uint64_t apart = (x > y ? x - y : y - x) % a_stride;
    return apart < width || a_stride - apart < width;
}

// Query-shaped rows [rows][heads x head_dim] of 16-bit numbers.
inline jfb_status check_rows(const char * what, const void * x, uint64_t stride, uint32_t rows, uint32_t heads,
                             const jfb_paged_cache & c) {
    if ((x == nullptr && rows > 0) || (reinterpret_cast<uintptr_t>(x) & 15u) != 0) {
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
