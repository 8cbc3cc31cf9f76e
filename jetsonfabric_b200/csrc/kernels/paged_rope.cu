// Rotary positions of q and k and the append of k and v to a cache in pages.
//
// A pair (x0, x1) at angle a = pos * freq becomes
//     y0 = (x0 cos a - x1 sin a) * factor,  y1 = (x0 sin a + x1 cos a) * factor.
// Angles of far positions lose all their digits in f32 (65536 rad has an ulp
// of 2^-7), so the angle's turns are formed and reduced in double, once per
// (row, pair), and shared by all heads through shared memory; the rotation is
// f32, each output rounded once.
//
// The kernel moves bytes: (q + k + v) in, the same out. A CTA takes 4 rows
// (one when few rows would leave SMs idle), its threads 16 elements at a time
// as 16-byte vectors: both partners of 8 pairs (half layout) or two 8-element
// runs. Rows or rotations that are not made of 8-element runs take the
// element-wise form of the same kernel.
#include <cmath>

#include "paged.cuh"

namespace jfb {
namespace paged {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 64;
constexpr int kMaxRows = 4;
constexpr uint64_t kNoSlot = ~0ull;

struct RopeParams {
    View view;
    const void * q;
    const void * k;
    const void * v;
    uint64_t q_stride, k_stride, v_stride, q_out_stride;
    const int32_t * pos;
    const double * freq;
    void * q_out;
    void * k_pool;
    void * v_pool;
    uint32_t heads, rope_dims, rows_per_cta;
    float factor;
};

template <typename S>
__device__ __forceinline__ float load1(const S * p);
template <>
__device__ __forceinline__ float load1<float>(const float * p) { return *p; }
template <>
__device__ __forceinline__ float load1<__half>(const __half * p) { return __half2float(*p); }
template <>
__device__ __forceinline__ float load1<__nv_bfloat16>(const __nv_bfloat16 * p) { return __bfloat162float(*p); }

template <typename T>
__device__ __forceinline__ T to16(float x);
template <>
__device__ __forceinline__ __half to16<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 to16<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename S>
__device__ __forceinline__ void load8(const S * p, float (&x)[8]) {
    if constexpr (sizeof(S) == 4) {
        const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = Num<S>::unpack(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

template <typename T>
__device__ __forceinline__ void store8(T * p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(Num<T>::pack(x[0], x[1]), Num<T>::pack(x[2], x[3]),
                                              Num<T>::pack(x[4], x[5]), Num<T>::pack(x[6], x[7]));
}

// One item of a head: the elements it covers, rotated or passed through.
// Vector form, half layout: items [0, P/8) are the pairs 8c .. 8c + 7, items
// behind them runs of 8 elements that pass through. Interleaved: runs of 8
// elements. Element-wise form: pairs, then single elements.
template <typename S, typename T, bool VEC, bool INTER>
__device__ __forceinline__ void rotate_item(const S * src, T * dst, uint32_t c, uint32_t pairs, const float2 * cs) {
    if constexpr (VEC && !INTER) {
        if (c < pairs / 8) {
            float a[8], b[8], y[8], z[8];
            load8(src + c * 8, a);
            load8(src + pairs + c * 8, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 t = cs[c * 8 + i];
                y[i] = a[i] * t.x - b[i] * t.y;
                z[i] = a[i] * t.y + b[i] * t.x;
            }
            store8(dst + c * 8, y);
            store8(dst + pairs + c * 8, z);
        } else {
            float a[8];
            const uint32_t at = 2 * pairs + (c - pairs / 8) * 8;
            load8(src + at, a);
            store8(dst + at, a);
        }
    } else if constexpr (VEC) {
        float a[8], y[8];
        load8(src + c * 8, a);
        if (c < pairs / 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 t = cs[c * 4 + i];
                y[2 * i] = a[2 * i] * t.x - a[2 * i + 1] * t.y;
                y[2 * i + 1] = a[2 * i] * t.y + a[2 * i + 1] * t.x;
            }
            store8(dst + c * 8, y);
        } else {
            store8(dst + c * 8, a);
        }
    } else {
        if (c < pairs) {
            const uint32_t i0 = INTER ? 2 * c : c, i1 = INTER ? 2 * c + 1 : c + pairs;
            const float a = load1(src + i0), b = load1(src + i1);
            dst[i0] = to16<T>(a * cs[c].x - b * cs[c].y);
            dst[i1] = to16<T>(a * cs[c].y + b * cs[c].x);
        } else {
            dst[c + pairs] = to16<T>(load1(src + c + pairs));
        }
    }
}

template <typename S, typename T, bool VEC, bool INTER>
__global__ void __launch_bounds__(kThreads) rope_append_kernel(const RopeParams p) {
    __shared__ float2 cs[kMaxRows][kMaxPairs];
    __shared__ uint64_t slot[kMaxRows];
    __shared__ uint32_t live[kMaxRows];
    pdl_trigger();
    pdl_wait();
    const View & v = p.view;
    const uint32_t row0 = blockIdx.x * p.rows_per_cta;
    const uint32_t rows = min(p.rows_per_cta, v.rows - row0);
    const uint32_t pairs = p.rope_dims / 2, hd = v.head_dim;
    for (uint32_t i = threadIdx.x; i < rows * pairs; i += kThreads) {
        const uint32_t r = i / pairs, j = i - r * pairs;
        // turns of the pair: only their fraction matters
        double turns = double(p.pos[row0 + r]) * p.freq[j] * 0.15915494309189533577;
        turns -= rint(turns);
        float s, c;
        sincospif(float(2.0 * turns), &s, &c);
        cs[r][j] = make_float2(c * p.factor, s * p.factor);
    }
    if (threadIdx.x < rows) {
        // the row's sequence, and where its key goes
        const uint32_t r = row0 + threadIdx.x;
        uint32_t lo = 0, hi = v.sequences;  // first b with q_start[b + 1] > r
        while (lo < hi) {
            const uint32_t mid = (lo + hi) / 2;
            if (v.q_start[mid + 1] > int32_t(r)) hi = mid;
            else lo = mid + 1;
        }
        uint64_t at = kNoSlot;
        bool in = lo < v.sequences;
        if (in) {
            const Sequence s = load_sequence(v, lo);
            in = r >= s.q0 && r - s.q0 < s.count;
            if (in) {
                const int64_t j = int64_t(s.kv) - s.count + (r - s.q0);
                const int32_t page = j < 0 ? -1 : v.table[uint64_t(lo) * v.table_stride + (uint64_t(j) >> v.page_shift)];
                if (page >= 0 && uint32_t(page) < v.pages) {
                    at = uint64_t(page) * v.page_stride + (uint64_t(j) & (v.page_size - 1)) * v.token_stride;
                } else {
                    flag_error(v.error, JFB_PAGED_ERROR_RANGE);
                }
            }
        }
        slot[threadIdx.x] = at;
        live[threadIdx.x] = in;
    }
    __syncthreads();
    const uint32_t per_head = VEC ? (INTER ? hd / 8 : hd / 8 - pairs / 8) : hd - pairs;
    const uint32_t v_head = VEC ? hd / 8 : hd;
    const uint32_t n_q = p.heads * per_head, n_k = v.kv_heads * per_head, n_v = v.kv_heads * v_head;
    for (uint32_t r = 0; r < rows; ++r) {
        if (!live[r]) continue;
        const uint64_t row = row0 + r, at = slot[r];
        for (uint32_t i = threadIdx.x; i < n_q + n_k + n_v; i += kThreads) {
            if (i < n_q) {
                const uint32_t h = i / per_head, c = i - h * per_head;
                rotate_item<S, T, VEC, INTER>(static_cast<const S *>(p.q) + row * p.q_stride + h * hd,
                                              static_cast<T *>(p.q_out) + row * p.q_out_stride + h * hd, c, pairs, cs[r]);
            } else if (at == kNoSlot) {
                break;
            } else if (i < n_q + n_k) {
                const uint32_t h = (i - n_q) / per_head, c = (i - n_q) - h * per_head;
                rotate_item<S, T, VEC, INTER>(static_cast<const S *>(p.k) + row * p.k_stride + h * hd,
                                              static_cast<T *>(p.k_pool) + at + h * v.head_stride, c, pairs, cs[r]);
            } else {
                const uint32_t h = (i - n_q - n_k) / v_head, c = (i - n_q - n_k) - h * v_head;
                const S * src = static_cast<const S *>(p.v) + row * p.v_stride + h * hd;
                T * dst = static_cast<T *>(p.v_pool) + at + h * v.head_stride;
                if constexpr (VEC) {
                    float x[8];
                    load8(src + c * 8, x);
                    store8(dst + c * 8, x);
                } else {
                    dst[c] = to16<T>(load1(src + c));
                }
            }
        }
    }
}

template <typename S, typename T>
cudaError_t launch(const RopeParams & p, bool vec, bool inter, cudaStream_t s) {
    const dim3 grid((p.view.rows + p.rows_per_cta - 1) / p.rows_per_cta), block(kThreads);
    if (vec) {
        return inter ? launch_k(rope_append_kernel<S, T, true, true>, grid, block, 0, s, p)
                     : launch_k(rope_append_kernel<S, T, true, false>, grid, block, 0, s, p);
    }
    return inter ? launch_k(rope_append_kernel<S, T, false, true>, grid, block, 0, s, p)
                 : launch_k(rope_append_kernel<S, T, false, false>, grid, block, 0, s, p);
}

bool aligned16(const void * x) { return (reinterpret_cast<uintptr_t>(x) & 15u) == 0; }

}  // namespace
}  // namespace paged
}  // namespace jfb

using namespace jfb;
using namespace jfb::paged;

extern "C" jfb_status jfb_rope_frequencies_host(double * freq, double * factor_out, uint32_t rope_dims, double base,
                                                uint32_t scaling, double factor, double trained, double low, double high) {
    if (freq == nullptr || factor_out == nullptr || rope_dims == 0 || rope_dims % 2 != 0 || !(base > 0.0) || !(base < 1e300)) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "rope frequencies need an even rope_dims and a positive base");
    }
    if (scaling > JFB_ROPE_SCALING_BANDS) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "unknown rope scaling %u", scaling);
    }
    if (scaling != JFB_ROPE_SCALING_NONE && !(factor >= 1.0 && factor < 1e30)) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "a rope scaling factor of at least 1 is required");
    }
    if (scaling >= JFB_ROPE_SCALING_YARN && !(trained > 0.0 && low > 0.0 && high > low)) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "this rope scaling needs a trained context and 0 < low < high");
    }
    if (scaling == JFB_ROPE_SCALING_YARN && base == 1.0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "YaRN needs a rope base other than 1");
    }
    if (scaling == JFB_ROPE_SCALING_NTK && rope_dims == 2) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "NTK-aware scaling needs more than one pair");
    }
    const double two_pi = 6.283185307179586476925, d = rope_dims;
    if (scaling == JFB_ROPE_SCALING_NTK) base *= std::pow(factor, d / (d - 2.0));
    // YaRN (Peng et al. 2023): the pair index at which a frequency makes `turns` turns over the trained context
    const auto index_of = [&](double turns) { return d * std::log(trained / (turns * two_pi)) / (2.0 * std::log(base)); };
    double from = 0.0, to = 1.0;
    if (scaling == JFB_ROPE_SCALING_YARN) {
        from = std::fmax(std::floor(index_of(high)), 0.0);
        to = std::fmin(std::ceil(index_of(low)), d - 1.0);
        if (to == from) to += 1e-3;
    }
    for (uint32_t i = 0; i < rope_dims / 2; ++i) {
        double f = std::pow(base, -2.0 * i / d);
        if (scaling == JFB_ROPE_SCALING_LINEAR) {
            f /= factor;
        } else if (scaling == JFB_ROPE_SCALING_YARN) {
            const double kept = 1.0 - std::fmin(std::fmax((i - from) / (to - from), 0.0), 1.0);
            f = f * kept + f / factor * (1.0 - kept);
        } else if (scaling == JFB_ROPE_SCALING_BANDS) {
            const double wave = two_pi / f;
            if (wave > trained / low) {
                f /= factor;
            } else if (wave > trained / high) {
                const double kept = (trained / wave - low) / (high - low);
                f = f * kept + f / factor * (1.0 - kept);
            }
        }
        freq[i] = f;
    }
    *factor_out = scaling == JFB_ROPE_SCALING_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
    return status_ok();
}

extern "C" jfb_status jfb_rope_paged_append(const void * q, const void * k, const void * v, uint32_t in_dtype,
                                            uint64_t q_stride, uint64_t k_stride, uint64_t v_stride, uint32_t rows,
                                            uint32_t heads, const int32_t * pos, const jfb_rope * rope,
                                            const jfb_paged_cache * cache, const jfb_paged_batch * batch, void * q_out,
                                            uint64_t q_out_stride, int32_t * error_flag, void * stream) {
    jfb_status st = check_cache(cache);
    if (st.code == JFB_STATUS_OK) st = check_batch(batch, true);
    if (st.code != JFB_STATUS_OK) return st;
    if (q == nullptr || k == nullptr || v == nullptr || pos == nullptr || q_out == nullptr || rope == nullptr ||
        rope->freq == nullptr) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_rope_paged_append operands are required");
    }
    if (in_dtype > JFB_DTYPE_BF16) return status_error(JFB_STATUS_INVALID_ARGUMENT, "unknown input dtype %u", in_dtype);
    const uint32_t hd = cache->head_dim, dims = rope->rope_dims;
    if (heads == 0 || heads > 65535u || dims < 2 || dims % 2 != 0 || dims > hd) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_rope_paged_append dimensions are inconsistent");
    }
    const uint64_t kv_row = uint64_t(cache->kv_heads) * hd, q_row = uint64_t(heads) * hd, most = 1ull << 40;
    if (q_stride < q_row || q_out_stride < q_row || k_stride < kv_row || v_stride < kv_row || q_stride >= most ||
        q_out_stride >= most || k_stride >= most || v_stride >= most) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_rope_paged_append row strides do not fit the heads");
    }
    if (q == q_out && (in_dtype != cache->dtype || q_stride != q_out_stride)) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "q in place needs the cache's dtype and one stride");
    }
    const uint32_t in_bytes = in_dtype == JFB_DTYPE_F32 ? 4 : 2;
    const uintptr_t natural = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
    if (natural % in_bytes != 0 || reinterpret_cast<uintptr_t>(q_out) % 2 != 0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_rope_paged_append operands are not aligned to their type");
    }
    if (rows > 0x7fffffffu) return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_rope_paged_append: too many rows");
    if (rows == 0 || batch->sequences == 0) return status_ok();
    RopeParams p;
    p.view = make_view(*cache, *batch, rows, 1, 0, error_flag);
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.q_out_stride = q_out_stride;
    p.pos = pos;
    p.freq = rope->freq;
    p.q_out = q_out;
    p.k_pool = cache->k;
    p.v_pool = cache->v;
    p.heads = heads;
    p.rope_dims = dims;
    p.factor = rope->factor;
    // fewer than about eight CTAs per SM with 4 rows each: one row per CTA
    p.rows_per_cta = rows >= 8u * 148u * kMaxRows ? kMaxRows : 1;
    const bool inter = rope->interleaved != 0;
    // 16-byte vectors: runs of 8 elements on both sides of every pair, aligned rows
    const bool vec = (inter ? dims % 8 == 0 : dims % 16 == 0) && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) &&
                     (q_stride | k_stride | v_stride | q_out_stride) % 8 == 0;
    cudaStream_t s = as_stream(stream);
    const bool half = cache->dtype == JFB_DTYPE_F16;
    cudaError_t e;
    if (in_dtype == JFB_DTYPE_F32) e = half ? launch<float, __half>(p, vec, inter, s) : launch<float, __nv_bfloat16>(p, vec, inter, s);
    else if (in_dtype == JFB_DTYPE_F16) e = half ? launch<__half, __half>(p, vec, inter, s) : launch<__half, __nv_bfloat16>(p, vec, inter, s);
    else e = half ? launch<__nv_bfloat16, __half>(p, vec, inter, s) : launch<__nv_bfloat16, __nv_bfloat16>(p, vec, inter, s);
    if (e != cudaSuccess) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_rope_paged_append: %s", cudaGetErrorString(e));
    return launch_status("jfb_rope_paged_append");
}
