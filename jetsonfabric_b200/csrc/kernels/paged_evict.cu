// Eviction: each sequence is cut, kv head by kv head, to its last `recent`
// keys and the heaviest of the others, in their order (keeping the keys that
// gathered most attention weight: Zhang et al. 2023).
//
// 1. select: a CTA per (sequence, kv head) brings the masses into shared memory
//    and orders them as unsigned numbers. The threshold (the need-th largest) is
//    found two bits at a time by counting how many reach each of three
//    candidates: sixteen passes over registers (up to 16384 keys) with one
//    barrier each (fewer once the kept set is settled), whose cost does not
//    depend on how the masses are spread
//    (a histogram of digits in shared memory was slower: the usual few octaves
//    make its counters collide). A last pass in slot order
//    keeps all above it and the first of those that equal it, so ties fall to
//    the lowest slot and the result is exact.
// 2. move: K and V rows to their new slots. Out of place, every 32 rows of a
//    (sequence, head) are a CTA of their own (D = 128), a thread moving 32-byte
//    sectors (66 us for a batch of 32 sequences of 1500 to 8192 keys cut to 2048,
//    4 kv heads, both steps; 75 with 16 bytes a thread). In place a CTA
//    owns a column slice of one (sequence, head) and walks the rows in order,
//    reading a whole step before it writes it: a row only moves to lower
//    slots, so a step overwrites no later step's source. The order costs time:
//    131 us for that batch, both steps.
#include <algorithm>

#include "paged.cuh"

namespace jfb {
namespace paged {
namespace {

constexpr uint32_t kCached = 49152;  // masses that fit shared memory
constexpr uint32_t kOwn = 16;        // keys a thread of the selection holds
// threads of the move and the pieces in flight in each
constexpr int kFarThreads = 128, kFarPieces = 2;
constexpr int kNearThreads = 512, kNearPieces = 8;

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
    uint32_t slices;  // columns of the move in place
    uint32_t cached;  // masses that the selection's shared memory holds
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

template <int kThreads>
__global__ void __launch_bounds__(kThreads) select_kernel(const EvictParams p) {
    constexpr uint32_t kWarps = kThreads / 32;
    extern __shared__ float cache[];
    __shared__ uint32_t counts[2][3][kWarps];
    __shared__ uint32_t above_of[kWarps], equal_of[kWarps];
    pdl_trigger();
    pdl_wait();
    const uint32_t b = blockIdx.x / p.view.kv_heads, t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const uint32_t len = evict_length(p, b);
    const float * mass = p.mass + uint64_t(blockIdx.x) * p.mass_stride;
    float * mass_out = p.mass_out + uint64_t(blockIdx.x) * p.mass_out_stride;
    int32_t * keep = p.keep + uint64_t(blockIdx.x) * p.budget;
    const uint32_t kept = min(len, p.budget);
    for (uint32_t i = kept + t; i < p.budget; i += kThreads) keep[i] = -1;
    if (len <= p.budget) {
        for (uint32_t i = t; i < len; i += kThreads) {
            keep[i] = int32_t(i);
            mass_out[i] = mass[i];
        }
        return;
    }
    const bool cached = len <= p.cached;
    if (cached) {
#pragma unroll 8
        for (uint32_t i = t; i < len; i += kThreads) cache[i] = mass[i];
    }
    __syncthreads();
    const auto mass_of = [&](uint32_t j) { return cached ? cache[j] : mass[j]; };
    const uint32_t tail = len - p.recent;  // from here on every slot is kept
    const uint32_t need = p.budget - p.recent;
    if (need > 0) {
        // the need-th largest of slots [0, tail): need < tail
        const bool own = cached && tail <= kOwn * kThreads;
        uint32_t keys[kOwn];  // 0 reaches no candidate
#pragma unroll
        for (uint32_t i = 0; i < kOwn; ++i) {
            const uint32_t j = t + i * kThreads;
            keys[i] = own && j < tail ? order_key(cache[j]) : 0u;
        }
        uint32_t threshold = 0, above = 0, reach = tail;  // how many exceed it, and how many reach it
        for (int shift = 30; shift >= 0; shift -= 2) {
            const uint32_t c1 = threshold | (1u << shift), c2 = threshold | (2u << shift), c3 = threshold | (3u << shift);
            uint32_t n1 = 0, n2 = 0, n3 = 0;
            const uint32_t half = (shift >> 1) & 1;  // the other half is still read by who is a pass behind
            if (own) {
                // three counts of up to 512 a warp in one word, then two of up to 16384 in another
                uint32_t n = 0;
#pragma unroll
                for (uint32_t i = 0; i < kOwn; ++i) {
                    if (i * kThreads < tail) {
                        n += keys[i] >= c1 ? 1u : 0u;
                        n += keys[i] >= c2 ? 1u << 10 : 0u;
                        n += keys[i] >= c3 ? 1u << 20 : 0u;
                    }
                }
                n = __reduce_add_sync(0xffffffffu, n);
                if (lane == 0) counts[half][0][warp] = n;
                __syncthreads();
                n = lane < kWarps ? counts[half][0][lane] : 0u;
                const uint32_t low = __reduce_add_sync(0xffffffffu, (n & 1023u) | ((n >> 10) & 1023u) << 16);
                n1 = low & 0xffffu;
                n2 = low >> 16;
                n3 = __reduce_add_sync(0xffffffffu, n >> 20);
            } else {
                for (uint32_t j = t; j < tail; j += kThreads) {
                    const uint32_t k = order_key(mass_of(j));
                    n1 += k >= c1;
                    n2 += k >= c2;
                    n3 += k >= c3;
                }
                n1 = __reduce_add_sync(0xffffffffu, n1);
                n2 = __reduce_add_sync(0xffffffffu, n2);
                n3 = __reduce_add_sync(0xffffffffu, n3);
                if (lane == 0) {
                    counts[half][0][warp] = n1;
                    counts[half][1][warp] = n2;
                    counts[half][2][warp] = n3;
                }
                __syncthreads();
                n1 = __reduce_add_sync(0xffffffffu, lane < kWarps ? counts[half][0][lane] : 0u);
                n2 = __reduce_add_sync(0xffffffffu, lane < kWarps ? counts[half][1][lane] : 0u);
                n3 = __reduce_add_sync(0xffffffffu, lane < kWarps ? counts[half][2][lane] : 0u);
            }
            const uint32_t digit = n3 >= need ? 3u : n2 >= need ? 2u : n1 >= need ? 1u : 0u;
            if (digit < 3) above = digit == 2 ? n3 : digit == 1 ? n2 : n1;
            if (digit > 0) reach = digit == 3 ? n3 : digit == 2 ? n2 : n1;
            threshold |= digit << shift;
            if (reach == need) {  // those are the ones: nothing left to tell apart
                --threshold;
                above = need;
                break;
            }
        }
        // keep everything above the threshold and the first `ties` that equal it: a warp per run of slots
        const uint32_t ties = need - above;
        const uint32_t run = (tail + kThreads - 1) / kThreads * 32, begin = min(tail, warp * run), end = min(tail, begin + run);
        uint32_t na = 0, ne = 0;
        for (uint32_t j = begin + lane; j < end; j += 32) {
            const uint32_t k = order_key(mass_of(j));
            na += k > threshold;
            ne += k == threshold;
        }
        na = __reduce_add_sync(0xffffffffu, na);
        ne = __reduce_add_sync(0xffffffffu, ne);
        if (lane == 0) {
            above_of[warp] = na;
            equal_of[warp] = ne;
        }
        __syncthreads();
        na = __reduce_add_sync(0xffffffffu, lane < warp ? above_of[lane] : 0u);  // before this run
        ne = __reduce_add_sync(0xffffffffu, lane < warp ? equal_of[lane] : 0u);
        const uint32_t below = (1u << lane) - 1u;
        for (uint32_t base = begin; base < end; base += 32) {
            const uint32_t j = base + lane;
            const float x = j < end ? mass_of(j) : 0.0f;
            const uint32_t k = order_key(x);
            const uint32_t va = __ballot_sync(0xffffffffu, j < end && k > threshold);
            const uint32_t ve = __ballot_sync(0xffffffffu, j < end && k == threshold);
            const uint32_t a = na + __popc(va & below), e = ne + __popc(ve & below);
            if (((va >> lane) & 1u) != 0 || (((ve >> lane) & 1u) != 0 && e < ties)) {
                const uint32_t at = a + min(e, ties);
                keep[at] = int32_t(j);
                if (cached) mass_out[at] = x;
            }
            na += __popc(va);
            ne += __popc(ve);
        }
    }
    for (uint32_t j = tail + t; j < len; j += kThreads) {
        keep[need + (j - tail)] = int32_t(j);
        if (cached) mass_out[need + (j - tail)] = cache[j];
    }
    if (!cached) {
        // the masses in order, each step read before it is written: they may move in place
        __syncthreads();
        for (uint32_t base = 0; base < kept; base += kThreads) {
            const float x = base + t < kept ? mass[keep[base + t]] : 0.0f;
            __syncthreads();
            if (base + t < kept) mass_out[base + t] = x;
            __syncthreads();
        }
    }
}

// What a thread moves at once: 16 bytes, or a 32-byte sector.
struct Piece16 {
    static constexpr uint32_t kElements = 8;
    uint4 x;
    __device__ __forceinline__ void load(const uint16_t * p) { x = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void store(uint16_t * p) const { *reinterpret_cast<uint4 *>(p) = x; }
};
struct Piece32 {
    static constexpr uint32_t kElements = 16;
    uint32_t x[8];
    __device__ __forceinline__ void load(const uint16_t * p) {
        asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7])
                     : "l"(p)
                     : "memory");
    }
    __device__ __forceinline__ void store(uint16_t * p) const {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]),
                     "r"(x[5]), "r"(x[6]), "r"(x[7])
                     : "memory");
    }
};

template <class Piece, int THREADS, int PIECES, bool IN_PLACE>
__global__ void __launch_bounds__(THREADS) move_kernel(const EvictParams p) {
    pdl_trigger();
    pdl_wait();
    const View & v = p.view;
    const uint32_t line = blockIdx.x >> 1, b = line / v.kv_heads, head = line - b * v.kv_heads;
    uint16_t * pool = static_cast<uint16_t *>((blockIdx.x & 1) ? p.v : p.k);
    const int32_t * keep = p.keep + uint64_t(line) * p.budget;
    const int32_t * from = v.table + uint64_t(b) * v.table_stride;
    const int32_t * to = p.table_out + uint64_t(b) * p.table_out_stride;
    const uint32_t width = v.head_dim / Piece::kElements / p.slices, first = blockIdx.z * width;  // pieces of a row
    const uint32_t step = THREADS * PIECES / width;                                  // rows read before they are written
    const uint32_t kept = min(evict_length(p, b), p.budget);
    // Out of place the CTAs move in no order: through a copy of the batch's own
    // table they would read what others wrote. Its first page tells (every row's
    // page would cost 3 us of 65).
    const bool copied = !IN_PLACE && to[0] == from[0];
    // The new length may replace the old one that other CTAs still read: they
    // cut either to the same number of rows.
    if (head == 0 && (blockIdx.x & 1) == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) p.kv_len_out[b] = int32_t(kept);
    for (uint32_t row0 = blockIdx.y * step; row0 < kept; row0 += gridDim.y * step) {  // in place there is one y
        Piece x[PIECES];
        uint64_t dst[PIECES];
#pragma unroll
        for (int u = 0; u < PIECES; ++u) {
            const uint32_t i = threadIdx.x + u * THREADS, r = i / width, c = (first + i - r * width) * Piece::kElements;
            dst[u] = ~0ull;
            if (r < step && row0 + r < kept) {
                const uint32_t at = row0 + r;
                const uint32_t j = uint32_t(keep[at]);
                const int32_t src_page = from[j >> v.page_shift], dst_page = to[at >> v.page_shift];
                if (src_page >= 0 && uint32_t(src_page) < v.pages && dst_page >= 0 && uint32_t(dst_page) < v.pages) {
                    const uint64_t in = uint64_t(head) * v.head_stride + c;
                    dst[u] = uint64_t(dst_page) * v.page_stride + (at & (v.page_size - 1)) * v.token_stride + in;
                    const uint64_t src = uint64_t(src_page) * v.page_stride + (j & (v.page_size - 1)) * v.token_stride + in;
                    if (src == dst[u] || copied) {
                        if (src != dst[u]) flag_error(v.error, JFB_PAGED_ERROR_RANGE);
                        dst[u] = ~0ull;  // stays where it is
                    } else {
                        x[u].load(pool + src);
                    }
                } else {
                    flag_error(v.error, JFB_PAGED_ERROR_RANGE);
                }
            }
        }
        if (IN_PLACE) __syncthreads();
#pragma unroll
        for (int u = 0; u < PIECES; ++u) {
            if (dst[u] != ~0ull) x[u].store(pool + dst[u]);
        }
        if (IN_PLACE) __syncthreads();
    }
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
    if (batch->sequences > 0 &&
        (mass == nullptr || keep == nullptr || kv_len_out == nullptr || mass_out == nullptr || page_table_out == nullptr)) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict operands are required");
    }
    if (budget == 0 || recent > budget || budget > 0x7fffffffu) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict needs a budget of at least one and recent <= budget");
    }
    if (mass_stride == 0 || mass_out_stride < budget || table_out_stride < table_out_width ||
        uint64_t(table_out_width) * cache->page_size < budget) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict: mass_out or page_table_out does not hold %u keys", budget);
    }
    if (batch->sequences == 0) return status_ok();
    if (mass_out == mass && mass_out_stride != mass_stride) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict: mass in place needs one stride");
    }
    if (page_table_out == batch->page_table && table_out_stride != batch->table_stride) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict: a page table in place needs one stride");
    }
    if (uint64_t(batch->sequences) * cache->kv_heads > 0x3fffffffull) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_evict: too many sequences and heads");
    }
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
    p.cached = mass_stride < kCached ? uint32_t(mass_stride) : kCached;
    const bool in_place = page_table_out == batch->page_table;
    const uint32_t lines = batch->sequences * cache->kv_heads;
    const uint32_t pieces = cache->head_dim / 8;
    // in place: column slices of at least 64 bytes (DRAM's granularity) while the CTAs do not fill the SMs four times
    const Device device = current_device();
    p.slices = 1;
    while (in_place && p.slices < 4 && pieces % (p.slices * 2) == 0 && pieces / (p.slices * 2) >= 4 && lines * 2 * p.slices < 4 * device.sms) {
        p.slices *= 2;
    }
    // out of place in 32-byte sectors where rows are made of them
    const bool sectors = !in_place && cache->head_dim % 16 == 0 && (cache->page_stride | cache->token_stride | cache->head_stride) % 16 == 0 &&
                         ((reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v)) & 31u) == 0;
    const uint32_t step = kFarThreads * kFarPieces / (sectors ? pieces / 2 : pieces);
    // a CTA for every step of the rows that a sequence can keep, as far as the grid goes
    const uint64_t most = std::min({uint64_t(budget), uint64_t(batch->table_width) * cache->page_size, mass_stride});
    const uint32_t steps = in_place ? 1u : uint32_t(std::min<uint64_t>((most + step - 1) / step, 65535u));
    cudaStream_t s = as_stream(stream);
    // Short lines: a small CTA, whose barriers are cheaper (one sequence of 700
    // keys, 2 kv heads: 8.7 us with both steps, 10.5 with 1024 threads). The host
    // knows only how many masses a line can hold.
    cudaError_t e;
    if (p.cached <= kOwn * 256) {
        e = launch_k(select_kernel<256>, dim3(lines), dim3(256), p.cached * sizeof(float), s, p);
    } else {
        e = allow_smem<select_kernel<1024>>(device, kCached * sizeof(float));
        if (e == cudaSuccess) e = launch_k(select_kernel<1024>, dim3(lines), dim3(1024), p.cached * sizeof(float), s, p);
    }
    if (e == cudaSuccess) {
        e = in_place  ? launch_k(move_kernel<Piece16, kNearThreads, kNearPieces, true>, dim3(lines * 2, 1, p.slices), dim3(kNearThreads), 0, s, p)
            : sectors ? launch_k(move_kernel<Piece32, kFarThreads, kFarPieces, false>, dim3(lines * 2, steps), dim3(kFarThreads), 0, s, p)
                      : launch_k(move_kernel<Piece16, kFarThreads, kFarPieces, false>, dim3(lines * 2, steps), dim3(kFarThreads), 0, s, p);
    }
    if (e != cudaSuccess) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_evict: %s", cudaGetErrorString(e));
    return launch_status("jfb_paged_evict");
}
