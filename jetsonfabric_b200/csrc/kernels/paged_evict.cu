// Eviction: each sequence is cut, kv head by kv head, to its last `recent`
// keys and the heaviest of the others, in their order.
//
// 1. select: a CTA per (sequence, kv head). The keys' masses become unsigned
//    numbers that order like the floats; four passes over 8-bit digits find
//    the threshold (the need-th largest), a last pass in slot order keeps all
//    above it and the first of those that equal it, so ties fall to the lowest
//    slot and the result is exact. The masses stay in L1/L2 between passes.
// 2. move: K and V rows to their new slots, 16 bytes a thread, 8 in flight.
//    Out of place, every (row range, sequence, head) is its own CTA. In place
//    a CTA owns a column slice of one (sequence, head) and walks the rows in
//    order, reading a whole step before it writes it: a row only moves to
//    lower slots, so a step overwrites no later step's source.
#include "paged.cuh"

namespace jfb {
namespace paged {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kPieces = 8;  // 16-byte pieces in flight per thread of the move

struct EvictParams {
    View view;
    const float * mass;
    float * mass_out;
    int32_t * keep;
    int32_t * kv_len_out;
    const int32_t * table_out;
    void * k;
    void * v;
    uint64_t mass_stride, mass_out_stride, table_out_stride;
    uint32_t budget, recent;
    uint32_t slices, row_steps;  // of the move's grid
    bool in_place;
};

// Unsigned numbers in the order of the floats; equal zeros, NaN least.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 becomes +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint32_t evict_length(const EvictParams & p, uint32_t b) {
    bool bad = false;
    uint32_t len = cut_length(p.view, p.view.kv_len[b], bad);
    if (len > p.mass_stride) {
        bad = true;
        len = uint32_t(p.mass_stride);
    }
    if (bad) flag_error(p.view.error, JFB_PAGED_ERROR_RANGE);
    return len;
}

__global__ void __launch_bounds__(kThreads) select_kernel(const EvictParams p) {
    __shared__ uint32_t hist[kWarps][256];
    __shared__ uint32_t digits[256];
    __shared__ uint32_t warp_above[kWarps], warp_equal[kWarps];
    __shared__ uint32_t found, rest;
    pdl_trigger();
    pdl_wait();
    const uint32_t b = blockIdx.x / p.view.kv_heads, t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const uint32_t len = evict_length(p, b);
    const float * mass = p.mass + uint64_t(blockIdx.x) * p.mass_stride;
    float * mass_out = p.mass_out + uint64_t(blockIdx.x) * p.mass_out_stride;
    int32_t * keep = p.keep + uint64_t(blockIdx.x) * p.budget;
    uint32_t done = 0;  // kept so far
    uint32_t tail = 0;  // from here on every slot is kept
    if (len > p.budget) {
        tail = len - p.recent;
        const uint32_t need = p.budget - p.recent;
        if (need > 0) {
            // the need-th largest of slots [0, tail): need <= budget - recent < tail
            uint32_t prefix = 0, left = need;
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (uint32_t i = t; i < kWarps * 256; i += kThreads) (&hist[0][0])[i] = 0;
                __syncthreads();
                const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
                for (uint32_t j = t; j < tail; j += kThreads) {
                    const uint32_t key = order_key(mass[j]);
                    if ((key & mask) == prefix) atomicAdd(&hist[warp][(key >> shift) & 255u], 1u);
                }
                __syncthreads();
                if (t < 256) {
                    uint32_t sum = 0;
                    for (int w = 0; w < kWarps; ++w) sum += hist[w][t];
                    digits[t] = sum;
                }
                __syncthreads();
                if (warp == 0) {
                    // from the largest digit down: lane l holds digits 255 - 8l .. 248 - 8l
                    uint32_t mine = 0;
                    for (int i = 0; i < 8; ++i) mine += digits[255 - 8 * lane - i];
                    uint32_t upto = mine;
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) {
                        const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d);
                        if (int(lane) >= d) upto += o;
                    }
                    const uint32_t over = __ballot_sync(0xffffffffu, upto >= left);
                    if (int(lane) == __ffs(over) - 1) {
                        uint32_t r = left - (upto - mine);
                        uint32_t d = 255 - 8 * lane;
                        while (digits[d] < r) r -= digits[d--];
                        found = d;
                        rest = r;
                    }
                }
                __syncthreads();
                prefix |= found << shift;
                left = rest;
            }
            // keep everything above the threshold and its first `left` equals
            uint32_t equal_before = 0;
            for (uint32_t base = 0; base < tail; base += kThreads) {
                const uint32_t j = base + t;
                const float x = j < tail ? mass[j] : 0.0f;
                const uint32_t key = order_key(x);
                const bool above = j < tail && key > prefix, equal = j < tail && key == prefix;
                const uint32_t va = __ballot_sync(0xffffffffu, above), ve = __ballot_sync(0xffffffffu, equal);
                if (lane == 0) {
                    warp_above[warp] = __popc(va);
                    warp_equal[warp] = __popc(ve);
                }
                __syncthreads();
                uint32_t a = 0, e = 0, all_a = 0, all_e = 0;
                for (int w = 0; w < kWarps; ++w) {
                    const uint32_t ca = warp_above[w], ce = warp_equal[w];
                    if (w < int(warp)) a += ca, e += ce;
                    all_a += ca;
                    all_e += ce;
                }
                const uint32_t below = (1u << lane) - 1u;
                a += __popc(va & below);
                e += equal_before + __popc(ve & below);
                // kept before this slot: those above, and equals up to `left`
                if (above || (equal && e < left)) {
                    const uint32_t at = done + a + min(e, left) - min(equal_before, left);
                    keep[at] = int32_t(j);
                    mass_out[at] = x;
                }
                done += all_a + min(equal_before + all_e, left) - min(equal_before, left);
                equal_before += all_e;
                __syncthreads();
            }
        }
    }
    for (uint32_t base = tail; base < len; base += kThreads) {
        const uint32_t j = base + t;
        const float x = j < len ? mass[j] : 0.0f;
        __syncthreads();  // in place: read before anything behind it is written
        if (j < len) {
            keep[done + (j - tail)] = int32_t(j);
            mass_out[done + (j - tail)] = x;
        }
        __syncthreads();
    }
    for (uint32_t i = min(len, p.budget) + t; i < p.budget; i += kThreads) keep[i] = -1;
}

__global__ void __launch_bounds__(kThreads) move_kernel(const EvictParams p) {
    pdl_trigger();
    pdl_wait();
    const View & v = p.view;
    const uint32_t line = blockIdx.x >> 1, b = line / v.kv_heads, head = line % v.kv_heads;
    uint16_t * pool = static_cast<uint16_t *>((blockIdx.x & 1) ? p.v : p.k);
    const int32_t * keep = p.keep + uint64_t(line) * p.budget;
    const int32_t * from = v.table + uint64_t(b) * v.table_stride;
    const int32_t * to = p.table_out + uint64_t(b) * p.table_out_stride;
    const uint32_t width = v.head_dim / 8 / p.slices, first = blockIdx.y * width;  // pieces of a row
    const uint32_t step = kThreads * kPieces / width;                                // rows read before they are written
    const uint32_t len = evict_length(p, b);
    const uint32_t kept = min(len, p.budget);
    const uint32_t begin = p.in_place ? 0u : blockIdx.z * step, end = p.in_place ? kept : min(kept, begin + step);
    for (uint32_t row0 = begin; row0 < end; row0 += step) {
        uint4 x[kPieces];
        uint64_t dst[kPieces];
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            const uint32_t i = threadIdx.x + u * kThreads, r = i / width, c = (first + i - r * width) * 8;
            dst[u] = ~0ull;
            x[u] = make_uint4(0, 0, 0, 0);
            if (r < step && row0 + r < end) {
                const uint32_t at = row0 + r;
                const uint32_t j = uint32_t(keep[at]);
                const int32_t src_page = from[j >> v.page_shift], dst_page = to[at >> v.page_shift];
                if (src_page >= 0 && uint32_t(src_page) < v.pages && dst_page >= 0 && uint32_t(dst_page) < v.pages) {
                    const uint64_t in = uint64_t(head) * v.head_stride + c;
                    dst[u] = uint64_t(dst_page) * v.page_stride + (at & (v.page_size - 1)) * v.token_stride + in;
                    const uint64_t src = uint64_t(src_page) * v.page_stride + (j & (v.page_size - 1)) * v.token_stride + in;
                    if (src == dst[u]) dst[u] = ~0ull;  // stays where it is
                    else x[u] = *reinterpret_cast<const uint4 *>(pool + src);
                } else {
                    flag_error(v.error, JFB_PAGED_ERROR_RANGE);
                }
            }
        }
        if (p.in_place) __syncthreads();
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            if (dst[u] != ~0ull) *reinterpret_cast<uint4 *>(pool + dst[u]) = x[u];
        }
        if (p.in_place) __syncthreads();
    }
}

// The new lengths, written last: kv_len_out may be the batch's kv_len.
__global__ void __launch_bounds__(kThreads) length_kernel(const EvictParams p) {
    pdl_trigger();
    pdl_wait();
    const uint32_t b = blockIdx.x * kThreads + threadIdx.x;
    if (b < p.view.sequences) p.kv_len_out[b] = int32_t(min(evict_length(p, b), p.budget));
}

}  // namespace
}  // namespace paged
}  // namespace jfb

using namespace jfb;
using namespace jfb::paged;

extern "C" jfb_status jfb_paged_evict(const float * mass, uint64_t mass_stride, const jfb_paged_cache * cache,
                                      const jfb_paged_batch * batch, uint32_t budget, uint32_t recent, int32_t * keep,
                                      int32_t * kv_len_out, float * mass_out, uint64_t mass_out_stride,
                                      const int32_t * page_table_out, uint64_t table_out_stride, uint32_t table_out_width,
                                      int32_t * error_flag, void * stream) {
    jfb_status st = check_cache(cache);
    if (st.code == JFB_STATUS_OK) st = check_batch(batch, false);
    if (st.code != JFB_STATUS_OK) return st;
    if (mass == nullptr || keep == nullptr || kv_len_out == nullptr || mass_out == nullptr || page_table_out == nullptr) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict operands are required");
    }
    if (budget == 0 || recent > budget || budget > 0x7fffffffu) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict needs a budget of at least one and recent <= budget");
    }
    if (mass_stride == 0 || mass_out_stride < budget || table_out_stride < table_out_width ||
        uint64_t(table_out_width) * cache->page_size < budget) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict: mass_out or page_table_out does not hold %u keys", budget);
    }
    if (mass_out == mass && mass_out_stride != mass_stride) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict: mass in place needs one stride");
    }
    if (page_table_out == batch->page_table && table_out_stride != batch->table_stride) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict: a page table in place needs one stride");
    }
    if (uint64_t(batch->sequences) * cache->kv_heads > 0x3fffffffull) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict: too many sequences and heads");
    }
    if (batch->sequences == 0) return status_ok();
    EvictParams p;
    p.view = make_view(*cache, *batch, 0, 1, 0, error_flag);
    p.mass = mass;
    p.mass_out = mass_out;
    p.keep = keep;
    p.kv_len_out = kv_len_out;
    p.table_out = page_table_out;
    p.k = cache->k;
    p.v = cache->v;
    p.mass_stride = mass_stride;
    p.mass_out_stride = mass_out_stride;
    p.table_out_stride = table_out_stride;
    p.budget = budget;
    p.recent = recent;
    p.in_place = page_table_out == batch->page_table;
    // column slices of at least 64 bytes (DRAM's granularity) while in-place CTAs do not fill the SMs
    const uint32_t lines = batch->sequences * cache->kv_heads;
    const uint32_t pieces = cache->head_dim / 8;
    p.slices = 1;
    while (p.in_place && p.slices < 4 && pieces % (p.slices * 2) == 0 && pieces / (p.slices * 2) >= 4 && lines * 2 * p.slices < 4 * 148) {
        p.slices *= 2;
    }
    const uint32_t step = kThreads * kPieces / (pieces / p.slices);
    const uint32_t steps = p.in_place ? 1u : (budget + step - 1) / step;
    if (steps > 65535u) return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict: a budget of %u is too large", budget);
    p.row_steps = steps;
    cudaStream_t s = as_stream(stream);
    cudaError_t e = launch_k(select_kernel, dim3(lines), dim3(kThreads), 0, s, p);
    if (e == cudaSuccess) e = launch_k(move_kernel, dim3(lines * 2, p.slices, steps), dim3(kThreads), 0, s, p);
    if (e == cudaSuccess) e = launch_k(length_kernel, dim3((batch->sequences + kThreads - 1) / kThreads), dim3(kThreads), 0, s, p);
    if (e != cudaSuccess) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_evict: %s", cudaGetErrorString(e));
    return launch_status("jfb_paged_evict");
}
