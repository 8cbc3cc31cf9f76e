// The attention weight each cached key received:
//     mass[j] += sum over rows r that see j of exp(scale q_r.k_j - lse_r).
// The sum runs along the rows, so the keys are the stationary side: an item is
// one tile of 128 keys of one sequence and kv head, no two CTAs add to the
// same key, and the order of every sum is fixed.
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

constexpr int kConsumers = 8;
constexpr int kThreadsRows = (kConsumers + 1) * 32;

template <int D>
struct MassSmem {
    static constexpr int kStages = D == 128 ? 6 : 12;
    static constexpr uint32_t kBars = kStages * kTileBytes<D>;  // full, empty
    static constexpr uint32_t kWalk = kBars + 2 * kStages * 8;
    static constexpr uint32_t kFlags = kWalk + 64;
    static constexpr uint32_t kBytes = kFlags + 16 + 1024;
};

// Key tiles of all sequences in one line, kv head outermost, divided evenly.
struct KeyWalk {
    uint64_t unit, end;
    uint32_t kv_head, b, tile;
    Sequence s;
    uint32_t limit;  // keys of the sequence that are written
};

__device__ __forceinline__ uint32_t key_limit(const View & v, const Sequence & s, uint64_t mass_stride) {
    if (s.kv > mass_stride) {
        flag_error(v.error, JFB_PAGED_ERROR_RANGE);
        return uint32_t(mass_stride);
    }
    return s.kv;
}

__device__ bool key_walk_begin(const View & v, uint64_t mass_stride, uint32_t * cost, KeyWalk * out, KeyWalk & w) {
    for (uint32_t b = threadIdx.x; b < v.sequences; b += blockDim.x) {
        cost[b] = (key_limit(v, load_sequence(v, b), mass_stride) + kTileKeys - 1) / kTileKeys;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const uint32_t lane = threadIdx.x;
        unsigned long long per_head = 0;
        for (uint32_t b = lane; b < v.sequences; b += 32) per_head += cost[b];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) per_head += __shfl_xor_sync(0xffffffffu, per_head, d);
        const unsigned long long total = per_head * v.kv_heads;
        KeyWalk x;
        x.unit = total * blockIdx.x / gridDim.x;
        x.end = total * (blockIdx.x + 1) / gridDim.x;
        x.kv_head = x.b = x.tile = x.limit = 0;
        x.s = Sequence{0, 0, 0};
        if (x.unit < x.end) {
            x.kv_head = uint32_t(x.unit / per_head);
            unsigned long long left = x.unit - per_head * x.kv_head;
            for (uint32_t base = 0; base < v.sequences; base += 32) {
                const unsigned long long mine = base + lane < v.sequences ? cost[base + lane] : 0u;
                unsigned long long upto = mine;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const unsigned long long o = __shfl_up_sync(0xffffffffu, upto, d);
                    if (int(lane) >= d) upto += o;
                }
                const uint32_t over = __ballot_sync(0xffffffffu, upto > left);
                if (over != 0) {
                    const int src = __ffs(over) - 1;
                    x.b = base + src;
                    left -= __shfl_sync(0xffffffffu, upto - mine, src);
                    break;
                }
                left -= __shfl_sync(0xffffffffu, upto, 31);
            }
            x.tile = uint32_t(left);
            x.s = load_sequence(v, x.b);
            x.limit = key_limit(v, x.s, mass_stride);
        }
        if (lane == 0) *out = x;
    }
    __syncthreads();
    w = *out;
    __syncthreads();
    return w.unit < w.end;
}

__device__ __forceinline__ bool key_walk_next(const View & v, uint64_t mass_stride, KeyWalk & w) {
    if (++w.unit >= w.end) return false;
    ++w.tile;
    while (uint64_t(w.tile) * kTileKeys >= w.limit) {
        w.tile = 0;
        if (++w.b >= v.sequences) {
            w.b = 0;
            ++w.kv_head;
        }
        w.s = load_sequence(v, w.b);
        w.limit = key_limit(v, w.s, mass_stride);
    }
    return true;
}

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
    static_assert(L::kBars >= JFB_PAGED_MAX_SEQUENCES * 4 && sizeof(KeyWalk) <= 64);
    uint8_t * smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t * full = reinterpret_cast<uint64_t *>(smem + L::kBars);
    uint64_t * empty = full + L::kStages;
    volatile int * flags = reinterpret_cast<volatile int *>(smem + L::kFlags);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, kConsumers);
        }
        flags[0] = 0;
        mbar_init_fence();
    }
    pdl_trigger();
    pdl_wait();
    const View & v = p.view;
    KeyWalk w;
    if (!key_walk_begin(v, v.slots, reinterpret_cast<uint32_t *>(smem), reinterpret_cast<KeyWalk *>(smem + L::kWalk), w)) return;
    fence_proxy_async();  // the ring held the walk's scratch
    __syncthreads();

    if (warp == kConsumers) {
        uint32_t n = 0;
        bool ok = true;
        auto pages_of = [&](const KeyWalk & a) {
            const uint32_t key0 = a.tile * kTileKeys;
            return tile_pages(v, v.table + uint64_t(a.b) * v.table_stride, key0, min(a.limit, key0 + uint32_t(kTileKeys)));
        };
        TileLoad next = pages_of(w);
        for (bool more = true; more; ++n) {
            const TileLoad load = next;
            const uint32_t head = w.kv_head;
            more = key_walk_next(v, v.slots, w);
            if (more) next = pages_of(w);
            const uint32_t st = n % L::kStages, turn = n / L::kStages;
            if (turn > 0) ok = __all_sync(0xffffffffu, mbar_wait(empty + st, (turn - 1) & 1, flags, v.error));
            if (!ok) break;
            tile_issue<D>(load, &map_k, head, smem_u32(smem) + st * kTileBytes<D>, full + st);
        }
        if (flags[0]) {
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
        const uint32_t st = n % L::kStages, parity = (n / L::kStages) & 1;
        ++n;
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
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + st);
        const uint32_t key = w.tile * kTileKeys + warp * 16;
        if (key < w.limit) {
            const int64_t first = int64_t(w.s.kv) - w.s.count;
            uint32_t r0, r1;
            seeing_rows(w.s, G, v.window, key, min(w.limit, key + 16), r0, r1);
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (uint32_t base = r0; base < r1; base += 16) {
                float s[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
                }
                uint32_t qa[D / 16][4];
                float lse2[2];
                int32_t pos[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t r = base + grp + 8 * e;
                    const bool valid = r < r1;
                    const uint32_t i = valid ? r / G : 0u, h = w.kv_head * G + (valid ? r % G : 0u);
                    const T * src = static_cast<const T *>(p.q) + uint64_t(w.s.q0 + i) * p.q_stride + uint64_t(h) * hd;
                    lse2[e] = valid ? p.lse[uint64_t(w.s.q0 + i) * p.heads + h] * kLog2e : 0.0f;
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
                        if (seen) acc[j * 2 + (e & 1)] += exp2_approx(fmaf(s[j][e], scale2, -lse2[e >> 1]));
                    }
                }
            }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
#pragma unroll
                for (int x = 0; x < 4; ++x) acc[x] += __shfl_xor_sync(0xffffffffu, acc[x], d);
            }
            if (grp == 0) {
                const uint64_t line = (uint64_t(w.b) * v.kv_heads + w.kv_head) * v.slots;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint32_t k = key + (x >> 1) * 8 + tig * 2 + (x & 1);
                    if (k < w.limit) {
                        const float before = p.mass_in != nullptr && int64_t(k) < first ? p.mass_in[line + k] : 0.0f;
                        p.mass_out[line + k] = before + acc[x];
                    }
                }
            }
        }
    } while (key_walk_next(v, v.slots, w));
}

template <typename T, int D>
jfb_status launch_rows(const CUtensorMap & k, const MassParams & p, uint32_t sms, cudaStream_t s) {
    auto kernel = mass_rows_kernel<T, D>;
    cudaError_t e = allow_smem(kernel, MassSmem<D>::kBytes);
    if (e == cudaSuccess) e = launch_k(kernel, dim3(sms), dim3(kThreadsRows), MassSmem<D>::kBytes, s, k, p);
    if (e != cudaSuccess) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention_mass: %s", cudaGetErrorString(e));
    return launch_status("jfb_paged_attention_mass");
}

}  // namespace
}  // namespace paged
}  // namespace jfb

using namespace jfb;
using namespace jfb::paged;

extern "C" jfb_status jfb_paged_attention_mass(const void * q, uint64_t q_stride, uint32_t rows, uint32_t heads, float scale,
                                               uint32_t window, const float * lse, const jfb_paged_cache * cache,
                                               const jfb_paged_batch * batch, const float * mass_in, float * mass_out,
                                               uint64_t mass_stride, int32_t * error_flag, void * stream) {
    jfb_status st = check_cache(cache);
    if (st.code == JFB_STATUS_OK) st = check_batch(batch, true);
    if (st.code == JFB_STATUS_OK) st = check_rows("jfb_paged_attention_mass", q, q_stride, rows, heads, *cache);
    if (st.code != JFB_STATUS_OK) return st;
    if (lse == nullptr || mass_out == nullptr || mass_stride == 0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_attention_mass needs lse and mass_out");
    }
    if (!(scale > 0.0f) || scale > 3.0e38f || window > 0x7fffffffu) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT,
                            "jfb_paged_attention_mass needs a positive finite scale and a window below 2^31");
    }
    const uint32_t sms = device_sms();
    if (sms == 0) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention_mass: no usable device");
    if (batch->sequences == 0) return status_ok();
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
    const uint32_t group = p.view.group;
    if (group <= 128 && uint64_t(rows) * group > 32ull * batch->sequences) return launch_mass_tc(*cache, mk, p, sms, s);
    if (cache->head_dim <= 64) {
        return half ? launch_rows<__half, 64>(mk, p, sms, s) : launch_rows<__nv_bfloat16, 64>(mk, p, sms, s);
    }
    return half ? launch_rows<__half, 128>(mk, p, sms, s) : launch_rows<__nv_bfloat16, 128>(mk, p, sms, s);
}
