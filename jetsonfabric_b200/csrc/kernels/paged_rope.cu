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
// (one when few rows would leave SMs idle), its threads 16-byte vectors: both
// partners of 8 pairs (half layout) or a run of 8 elements. Sixteen small CTAs
// an SM keep more loads in flight than several items per thread did (2, 4 and 8
// of them: 63, 73 and 89 us against 55 for 16192 rows of 36 heads, bf16, 5.4
// TB/s). Rows or rotations that are not made of 8-element runs take an
// element-wise form.
#include <cmath>

#include "paged.cuh"

namespace jfb {
namespace paged {
namespace {

constexpr int kThreads = 128;
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

// Eight elements as they lie in memory.
template <typename S>
struct Raw8 {
    uint4 w[sizeof(S) / 2];
    __device__ __forceinline__ void load(const S * p) {
#pragma unroll
        for (int i = 0; i < int(sizeof(S)) / 2; ++i) w[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < int(sizeof(S)) / 2; ++i) {
            const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (sizeof(S) == 4) {
                    x[4 * i + k] = __uint_as_float(u[k]);
                } else {
                    const float2 f = Num<S>::unpack(u[k]);
                    x[2 * k] = f.x;
                    x[2 * k + 1] = f.y;
                }
            }
        }
    }
};

template <typename T>
__device__ __forceinline__ void store8(T * p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(Num<T>::pack(x[0], x[1]), Num<T>::pack(x[2], x[3]),
                                              Num<T>::pack(x[4], x[5]), Num<T>::pack(x[6], x[7]));
}

// Item c of a head in vectors. Half layout: items [0, P/8) are the pairs 8c ..
// 8c + 7, those behind them runs of 8 elements that pass through. Interleaved:
// runs of 8 elements. `turned` is false for v.
template <typename S, typename T, bool INTER>
struct VectorItem {
    T * dst;
    const float2 * cs;
    uint32_t pairs;  // distance of the partners; 0: one run
    Raw8<S> a, b;
    __device__ __forceinline__ void load(const S * src, T * to, uint32_t c, uint32_t half, bool turned, const float2 * turns) {
        if constexpr (INTER) {
            pairs = 0;
            cs = turned && c < half / 4 ? turns + c * 4 : nullptr;
            a.load(src + c * 8);
            dst = to + c * 8;
        } else {
            const bool both = turned && c < half / 8;
            const uint32_t at = both || !turned ? c * 8 : half + c * 8;
            pairs = both ? half : 0u;
            cs = turns + c * 8;
            a.load(src + at);
            if (both) b.load(src + half + c * 8);
            dst = to + at;
        }
    }
    __device__ __forceinline__ void store() const {
        float x[8], y[8];
        a.get(x);
        if constexpr (INTER) {
            if (cs != nullptr) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 t = cs[i];
                    const float x0 = x[2 * i], x1 = x[2 * i + 1];
                    x[2 * i] = x0 * t.x - x1 * t.y;
                    x[2 * i + 1] = x0 * t.y + x1 * t.x;
                }
            }
        } else if (pairs != 0) {
            b.get(y);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 t = cs[i];
                const float x0 = x[i], x1 = y[i];
                x[i] = x0 * t.x - x1 * t.y;
                y[i] = x0 * t.y + x1 * t.x;
            }
            store8(dst + pairs, y);
        }
        store8(dst, x);
    }
};

// The same in elements: pairs, then single elements that pass through.
template <typename S, typename T, bool INTER>
__device__ __forceinline__ void element_item(const S * src, T * dst, uint32_t c, uint32_t half, bool turned, const float2 * cs) {
    if (!turned) {
        dst[c] = to16<T>(load1(src + c));
    } else if (c < half) {
        const uint32_t i0 = INTER ? 2 * c : c, i1 = INTER ? 2 * c + 1 : c + half;
        const float a = load1(src + i0), b = load1(src + i1);
        dst[i0] = to16<T>(a * cs[c].x - b * cs[c].y);
        dst[i1] = to16<T>(a * cs[c].y + b * cs[c].x);
    } else {
        dst[c + half] = to16<T>(load1(src + c + half));
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
                // from the length as it is, not as the table cuts it: that slot holds another key
                const int64_t j = int64_t(v.kv_len[lo]) - s.count + (r - s.q0);
                const bool there = j >= 0 && j < int64_t(capacity(v));
                const int32_t page = there ? v.table[uint64_t(lo) * v.table_stride + (uint64_t(j) >> v.page_shift)] : -1;
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
    const uint32_t n_q = p.heads * per_head, n_k = v.kv_heads * per_head, n_row = n_q + n_k + v.kv_heads * v_head;
    // source, destination and place in its head of item i of the CTA's rows; no destination: nothing to do
    struct Place {
        const S * src;
        T * dst;
        uint32_t c, r;
        bool turned;
    };
    const auto place = [&](uint32_t i) {
        Place o;
        o.r = i / n_row;
        i -= o.r * n_row;
        const uint64_t row = row0 + o.r, at = slot[o.r];
        o.turned = i < n_q + n_k;
        if (i < n_q) {
            const uint32_t h = i / per_head;
            o.c = i - h * per_head;
            o.src = static_cast<const S *>(p.q) + row * p.q_stride + h * hd;
            o.dst = static_cast<T *>(p.q_out) + row * p.q_out_stride + h * hd;
        } else if (o.turned) {
            const uint32_t h = (i - n_q) / per_head;
            o.c = (i - n_q) - h * per_head;
            o.src = static_cast<const S *>(p.k) + row * p.k_stride + h * hd;
            o.dst = at == kNoSlot ? nullptr : static_cast<T *>(p.k_pool) + at + h * v.head_stride;
        } else {
            const uint32_t h = (i - n_q - n_k) / v_head;
            o.c = (i - n_q - n_k) - h * v_head;
            o.src = static_cast<const S *>(p.v) + row * p.v_stride + h * hd;
            o.dst = at == kNoSlot ? nullptr : static_cast<T *>(p.v_pool) + at + h * v.head_stride;
        }
        if (!live[o.r]) o.dst = nullptr;
        return o;
    };
    const uint32_t total = rows * n_row;
    if constexpr (VEC) {
        for (uint32_t i = threadIdx.x; i < total; i += kThreads) {
            const Place o = place(i);
            if (o.dst == nullptr) continue;
            VectorItem<S, T, INTER> item;
            item.load(o.src, o.dst, o.c, pairs, o.turned, cs[o.r]);
            item.store();
        }
    } else {
        for (uint32_t i = threadIdx.x; i < total; i += kThreads) {
            const Place o = place(i);
            if (o.dst != nullptr) element_item<S, T, INTER>(o.src, o.dst, o.c, pairs, o.turned, cs[o.r]);
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
        // Cut to the pairs there are, the ramp from `high` (kept before it) to `low`
        // (divided behind it) must not turn round: where every pair makes more
        // turns than `high` or fewer than `low`, it lies behind or before them all.
        const double first = std::floor(index_of(high)), last = std::ceil(index_of(low));
        from = std::fmax(first, 0.0);
        to = std::fmin(last, d - 1.0);
        if (base > 1.0 && first > d - 1.0) {
            from = d;
            to = d + 1.0;
        } else if (base > 1.0 && last <= 0.0) {
            from = -2.0;
            to = -1.0;
        }
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
    if (rope == nullptr || rope->freq == nullptr ||
        (rows > 0 && (q == nullptr || k == nullptr || v == nullptr || pos == nullptr || q_out == nullptr))) {
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
    if (q == q_out && rows > 0 && (in_dtype != cache->dtype || q_stride != q_out_stride)) {
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
    // Few rows: one per CTA, to fill the SMs; many: four share the work of finding their sequences and angles, and leave
    // fewer threads idle where a row has few heads. One / four, in us, for 12/2 heads (f32 in), 28/4 (bf16), 40/8 (f32):
    // 1000 rows 6.8/8.8, 10.0/13.9, 13.1/19.5; 2000 10.2/12.3, 11.4/16.1, 19.9/24.5; 4000 14.7/14.6, 18.6/21.3, 33.0/37.1;
    // 6000 19.2/15.8, 25.7/28.0, 45.1/46.7; 8000 23.9/23.2, 32.2/31.3, 57.5/65.2; 16192 42.0/37.4, 56.1/56.4, 108/113.
    p.rows_per_cta = rows >= 8u * current_device().sms * kMaxRows ? kMaxRows : 1;
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
