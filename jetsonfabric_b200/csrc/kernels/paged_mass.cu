// The attention weight each cached key received:
//     mass[j] += sum over rows r that see j of exp(scale q_r.k_j - lse_r).
// The sum runs along the rows, so the keys are the stationary side: an item is
// one tile of 128 keys of one sequence and kv head, no two CTAs add to the
// same key, and the order of every sum is fixed.
#include <algorithm>

#include "paged.cuh"
#include "paged_attention.cuh"
#include "paged_mass.cuh"

namespace jfb {
namespace paged {
namespace {

// ---- few rows -----------------------------------------------------------------------
//
// The K bytes bound a decode step. A producer warp brings K tiles page by page
// through TMA, 6 (D = 128) of them in flight per SM; each of the 8 consumer
// warps keeps 16 keys of a tile in registers and takes the packed rows (token,
// head of the group) 16 at a time through mma.sync m16n8k16.
// 64 sequences of 1025 to 1280 keys, 28/4 heads: 22 us (54 % of the measured copy
// bandwidth), bound by the consumers' fragment loads and sums per tile.

constexpr int kConsumers = 8;
constexpr int kThreadsRows = (kConsumers + 2) * 32;  // and the producers of K and of the masses

// A sequence and kv head is one item, its key tiles the units.
struct SequenceItems {
    struct Part {
        uint32_t tiles;
    };
    static __device__ __forceinline__ uint32_t limit(const View & v, const Sequence & s) {
        if (s.kv <= v.slots) return s.kv;
        flag_error(v.error, JFB_PAGED_ERROR_RANGE);
        return uint32_t(v.slots);
    }
    static __device__ __forceinline__ uint32_t count(const View & v, const Sequence & s) { return s.kv > 0 ? 1 : 0; }
    static __device__ __forceinline__ Part part(const View & v, const Sequence & s, uint32_t) {
        return Part{(limit(v, s) + kTileKeys - 1) / kTileKeys};
    }
};
using SequenceWalk = WalkOf<SequenceItems>;

template <int D>
struct MassSmem {
    static constexpr int kStages = D == 128 ? 6 : 12;
    static constexpr uint32_t kBefore = kStages * kTileBytes<D>;             // [stages][128] masses
    static constexpr uint32_t kBars = kBefore + kStages * kTileKeys * 4;     // full, empty
    static constexpr uint32_t kWalk = kBars + 2 * kStages * 8;
    static constexpr uint32_t kFlags = kWalk + kThreadsRows / 32 * sizeof(SequenceWalk);
    static constexpr uint32_t kBytes = kFlags + 16 + 1024;
};

// Packed rows [r0, r1) that see some of keys [key0, key1).
__device__ __forceinline__ void seeing_rows(const Sequence & s, uint32_t group, uint32_t window, uint32_t key0, uint32_t key1,
                                            uint32_t & r0, uint32_t & r1) {
    const int64_t first = int64_t(s.kv) - s.count;
    const int64_t i0 = int64_t(key0) - first;  // first row at or behind key0
    int64_t i1 = s.count;
    if (window > 0 && int64_t(key1) - 1 + window - first < i1) i1 = int64_t(key1) - 1 + window - first;
    r0 = i0 > 0 ? uint32_t(i0 < int64_t(s.count) ? i0 : int64_t(s.count)) * group : 0u;
    r1 = i1 > 0 ? uint32_t(i1) * group : 0u;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreadsRows, 1)
    mass_rows_kernel(const __grid_constant__ CUtensorMap map_k, const MassParams p) {
    extern __shared__ uint8_t smem_raw[];
    using L = MassSmem<D>;
    static_assert(L::kBars >= JFB_PAGED_MAX_SEQUENCES * 8);
    uint8_t * smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t * full = reinterpret_cast<uint64_t *>(smem + L::kBars);
    uint64_t * empty = full + L::kStages;
    volatile int * flags = reinterpret_cast<volatile int *>(smem + L::kFlags);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(full + i, 33);  // the K copy's announcement, and every producer lane's masses
            mbar_init(empty + i, kConsumers);
        }
        flags[0] = 0;
        mbar_init_fence();
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    const View & v = p.view;
    SequenceWalk * walks = reinterpret_cast<SequenceWalk *>(smem + L::kWalk);
    if (!walk_begin<0>(v, reinterpret_cast<uint64_t *>(smem), walks)) return;
    SequenceWalk & w = walks[warp];

    if (warp >= kConsumers) {
        const bool keys = warp == kConsumers;
        uint32_t n = 0;
        bool ok = true;
        do {
            uint32_t t0, t1;
            walk_segment<0>(w, t0, t1);
            const int32_t * row = v.table + uint64_t(w.b) * v.table_stride;
            const uint32_t limit = SequenceItems::limit(v, w.s), head = w.kv_head;
            const int64_t first = int64_t(w.s.kv) - w.s.count;
            const uint64_t line = (uint64_t(w.b) * v.kv_heads + w.kv_head) * v.slots;
            auto pages_of = [&](uint32_t t) {
                return tile_pages(v, row, t * kTileKeys, min(limit, (t + 1) * uint32_t(kTileKeys)));
            };
            TileLoad next = {};
            if (keys) next = pages_of(t0);
            for (uint32_t t = t0; t < t1; ++t, ++n) {
                const TileLoad load = next;
                if (keys && t + 1 < t1) next = pages_of(t + 1);
                const uint32_t st = n % L::kStages, turn = n / L::kStages;
                if (turn > 0) ok = __all_sync(0xffffffffu, mbar_wait(empty + st, (turn - 1) & 1, flags, v.error));
                if (!ok) break;
                if (keys) {
                    tile_issue<D>(v, load, &map_k, head, smem_u32(smem) + st * kTileBytes<D>, full + st);
                    continue;
                }
                const uint32_t to = smem_u32(smem) + L::kBefore + st * (kTileKeys * 4);
#pragma unroll
                for (uint32_t j = 0; j < uint32_t(kTileKeys) / 32; ++j) {  // zeros for new slots and behind the keys
                    const uint32_t i = j * 32 + lane, k = t * kTileKeys + i;
                    const bool held = p.mass_in != nullptr && k < limit && int64_t(k) < first;
                    const float * src = held ? p.mass_in + line + k : p.mass_out;
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + i * 4), "l"(src), "r"(held ? 4u : 0u) : "memory");
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full + st)) : "memory");
            }
        } while (ok && walk_warp_next<0>(v, &w));
        asm volatile("cp.async.wait_all;" ::: "memory");
        if (keys && flags[0]) {
            for (uint32_t i = n > uint32_t(L::kStages) ? n - L::kStages : 0u; i < n; ++i) {
                mbar_drain(full + i % L::kStages, (i / L::kStages) & 1);
            }
        }
        return;
    }

    const uint32_t grp = lane >> 2, tig = lane & 3;
    const uint32_t G = v.group, hd = v.head_dim;
    const float scale2 = p.scale * kLog2e;
    uint32_t n = 0;
    do {
        uint32_t t0, t1;
        walk_segment<0>(w, t0, t1);
        const int64_t first = int64_t(w.s.kv) - w.s.count;
        const uint32_t limit = SequenceItems::limit(v, w.s);
        const uint64_t line = (uint64_t(w.b) * v.kv_heads + w.kv_head) * v.slots;
        // 16 packed rows as A fragments, their -lse and slots
        uint32_t qa[D / 16][4];
        float nlse[2];
        int32_t pos[2];
        const auto load_rows = [&](uint32_t base, uint32_t end) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t r = base + grp + 8 * e;
                const bool valid = r < end;
                const uint32_t i = valid ? r / G : 0u, h = w.kv_head * G + (valid ? r % G : 0u);
                const T * src = static_cast<const T *>(p.q) + uint64_t(w.s.q0 + i) * p.q_stride + uint64_t(h) * hd;
                nlse[e] = valid ? -kLog2e * p.lse[uint64_t(w.s.q0 + i) * p.heads + h] : 0.0f;
                pos[e] = valid ? int32_t(first + i) : -1;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t d = kk * 16 + x * 8;
                        qa[kk][e + 2 * x] = valid && d < hd ? *reinterpret_cast<const uint32_t *>(src + d + tig * 2) : 0u;
                    }
                }
            }
        };
        const uint32_t packed = w.s.count * G;
        const bool once = packed <= 16;  // all rows fit: fetched once for the segment's tiles
        if (once) load_rows(0, packed);
        for (uint32_t t = t0; t < t1; ++t, ++n) {
            const uint32_t st = n % L::kStages, parity = (n / L::kStages) & 1;
            if (!__all_sync(0xffffffffu, mbar_wait(full + st, parity, flags, v.error))) return;  // no barrier joins these warps
            // this warp's 16 keys as B fragments, then the stage is free
            uint32_t kb[D / 16][4];
            const uint32_t kbase = smem_u32(smem) + st * kTileBytes<D>;
            const uint32_t krow = warp * 16 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t chunk = kk * 2 + ((lane >> 3) & 1);
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                             : "=r"(kb[kk][0]), "=r"(kb[kk][1]), "=r"(kb[kk][2]), "=r"(kb[kk][3])
                             : "r"(kbase + (chunk >> 3) * (kTileKeys * 128) + krow * 128 + (((chunk & 7) ^ (krow & 7)) << 4))
                             : "memory");
            }
            const float before = reinterpret_cast<const float *>(smem + L::kBefore)[st * kTileKeys + warp * 16 + (lane & 15)];
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + st);
            const uint32_t key = t * kTileKeys + warp * 16;
            if (key >= limit) continue;
            uint32_t r0, r1;
            seeing_rows(w.s, G, v.window, key, min(limit, key + 16), r0, r1);
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t base = once ? 0u : r0; base < r1; base += 16) {
                if (!once) load_rows(base, r1);
                float s[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
                }
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    mma_16816<T>(s[0], qa[kk], kb[kk][0], kb[kk][1]);
                    mma_16816<T>(s[1], qa[kk], kb[kk][2], kb[kk][3]);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int32_t k = int32_t(key) + j * 8 + int32_t(tig) * 2 + (e & 1), q = pos[e >> 1];
                        const bool seen = k <= q && (v.window == 0 || k > q - int32_t(v.window));
                        if (seen) acc[j * 2 + (e & 1)] += exp2_approx(fmaf(s[j][e], scale2, nlse[e >> 1]));
                    }
                }
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[x] += __shfl_xor_sync(0xffffffffu, acc[x], d);
            }
            // key i's sum lies in lane i % 8 / 2, register i / 8 * 2 + i % 2
            float sum = 0.0f;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float y = __shfl_sync(0xffffffffu, acc[x], (lane & 7) >> 1);
                if ((lane >> 3) * 2 + (lane & 1) == uint32_t(x)) sum = y;
            }
            if (lane < 16 && key + lane < limit) p.mass_out[line + key + lane] = before + sum;
        }
    } while (walk_warp_next<0>(v, &w));
}

template <typename T, int D>
jfb_status launch_rows(const CUtensorMap & k, const MassParams & p, const Device & device, cudaStream_t s) {
    cudaError_t e = allow_smem<mass_rows_kernel<T, D>>(device, MassSmem<D>::kBytes);
    if (e == cudaSuccess) e = launch_k(mass_rows_kernel<T, D>, dim3(device.sms), dim3(kThreadsRows), MassSmem<D>::kBytes, s, k, p);
    if (e != cudaSuccess) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention_mass: %s", cudaGetErrorString(e));
    return launch_status("jfb_paged_attention_mass");
}

}  // namespace
}  // namespace paged
}  // namespace jfb

using namespace jfb;
using namespace jfb::paged;

// The tcgen05 kernel from 2 row tiles of 16 a sequence on, if there is work for
// it, counted in (16 rows, 128 keys) tiles of the keys that the table and the
// masses can hold. Rows kernel / tcgen05 kernel at 28/4 heads, in us: 64
// sequences of 1150 keys with 4, 8, 16 new tokens 58/84, 99/84, 185/85; 4 of 1000
// with 8, 16, 40: 11/14, 16/14 (896 tiles), 31/18; one of 1000 with 16, 48: 15/14, 35/14
// (672); one of 8000 with 4, 8, 16: 11/14 (504), 16/14 (1008), 26/14.
//
// As for the attention, the keys are those the arrays can hold and the rows
// those of the mean sequence: 63 single tokens (23 us by themselves) with a
// chunk of 220 over 8000 keys (35) take 2490 us here, where the chunk's rows go
// through each key tile 16 at a time on the one CTA that holds it; with one of
// 512 (58) 267 on the tcgen05 kernel.
extern "C" int jfb_paged_attention_mass_uses_tiles(uint32_t rows, uint32_t heads, const jfb_paged_cache * cache,
                                                   const jfb_paged_batch * batch, uint64_t mass_stride) {
    const uint32_t group = heads / cache->kv_heads;
    const uint64_t keys = std::min(uint64_t(batch->table_width) * cache->page_size, mass_stride);
    const double tiles = double((uint64_t(rows) * group + 15) / 16) * cache->kv_heads * double((keys + kTileKeys - 1) / kTileKeys);
    return group <= 128 && uint64_t(rows) * group > 32ull * batch->sequences && tiles > 700;
}

extern "C" jfb_status jfb_paged_attention_mass(const void * q, uint64_t q_stride, uint32_t rows, uint32_t heads, float scale,
                                               uint32_t window, const float * lse, const jfb_paged_cache * cache,
                                               const jfb_paged_batch * batch, const float * mass_in, float * mass_out,
                                               uint64_t mass_stride, int32_t * error_flag, void * stream) {
    jfb_status st = check_cache(cache);
    if (st.code == JFB_STATUS_OK) st = check_batch(batch, true);
    if (st.code == JFB_STATUS_OK) st = check_rows("jfb_paged_attention_mass", q, q_stride, rows, heads, *cache);
    if (st.code != JFB_STATUS_OK) return st;
    if ((lse == nullptr && rows > 0) || (mass_out == nullptr && batch->sequences > 0) || mass_stride == 0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_attention_mass needs lse and mass_out");
    }
    if (!(scale > 0.0f) || scale > 1.0e38f || window > 0x7fffffffu) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT,
                            "jfb_paged_attention_mass needs a positive scale up to 1e38 and a window below 2^31");
    }
    if (batch->sequences == 0) return status_ok();
    const Device device = current_device();
    if (device.sms == 0) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention_mass: no usable device");
    MassParams p;
    p.view = make_view(*cache, *batch, rows, heads / cache->kv_heads, window, error_flag);
    p.view.slots = mass_stride;
    p.q = q;
    p.lse = lse;
    p.mass_in = mass_in;
    p.mass_out = mass_out;
    p.q_stride = q_stride;
    p.heads = heads;
    p.scale = scale;
    CUtensorMap mk;
    if (!pool_map(mk, cache->k, *cache)) {
        return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention_mass: could not encode a TMA tensor map");
    }
    cudaStream_t s = as_stream(stream);
    const bool half = cache->dtype == JFB_DTYPE_F16;
    if (jfb_paged_attention_mass_uses_tiles(rows, heads, cache, batch, mass_stride)) return launch_mass_tc(*cache, mk, p, device, s);
    if (cache->head_dim <= 64) {
        return half ? launch_rows<__half, 64>(mk, p, device, s) : launch_rows<__nv_bfloat16, 64>(mk, p, device, s);
    }
    return half ? launch_rows<__half, 128>(mk, p, device, s) : launch_rows<__nv_bfloat16, 128>(mk, p, device, s);
}
