// Attention of a chunk of new tokens over a KV cache in pages.
//
// For row r of sequence b at slot p:  x_j = scale q.k_j over the slots j <= p
// (and j > p - window), out = sum_j e^(x_j - m) v_j / sum_j e^(x_j - m). One
// pass over the keys keeps a running maximum m and rescales the sums when it
// grows; parts of one row that were formed apart (warps, CTAs) are joined the
// same way.
#include <algorithm>

#include "paged.cuh"
#include "paged_attention.cuh"

namespace jfb {
namespace paged {
namespace {

// ---- few rows -----------------------------------------------------------------------
//
// Decode and short chunks: each item has 16 packed rows (token, head of the
// group), so the K and V bytes bound the time (4 D bytes per key for 4 D G
// flops) and the products run on mma.sync m16n8k16, whose 16 rows waste the
// least of them. Two producer warps bring K and V tiles of 128 keys page by
// page through TMA into a ring of 3 (D = 128: 192 KB, 128 KB or more in flight
// per SM); of the 8 consumer warps each takes 16 keys of every tile with its
// own running maximum and sums, so warps meet only at the end of an item's
// segment, in shared memory.

constexpr int kRowsM = 16;
constexpr int kItemRows = 0;  // units of an item's start and end
constexpr int kConsumers = 8;
constexpr int kThreadsRows = (kConsumers + 2) * 32;

template <int D>
struct RowsSmem {
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr uint32_t kStage = 2 * kTileBytes<D>;
    static constexpr uint32_t kMerge = kStages * kStage;                       // [8 warps][16 rows][64] f32
    static constexpr uint32_t kMl = kMerge + kConsumers * kRowsM * 64 * 4;     // [8][16] (m, l)
    static constexpr uint32_t kBars = kMl + kConsumers * kRowsM * 8;           // full K, full V, empty
    static constexpr uint32_t kWalk = kBars + 3 * kStages * 8;
    static constexpr uint32_t kFlags = kWalk + kThreadsRows / 32 * sizeof(Walk);  // abort, last
    static constexpr uint32_t kBytes = kFlags + 16 + 1024;                     // + alignment
};
static_assert(RowsSmem<128>::kBytes <= 232448 && RowsSmem<64>::kBytes <= 232448);
static_assert(RowsSmem<64>::kMerge >= JFB_PAGED_MAX_SEQUENCES * 8);

__device__ __forceinline__ void bar_consumers() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreadsRows, 1)
    paged_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttentionParams p) {
    extern __shared__ uint8_t smem_raw[];
    using L = RowsSmem<D>;
    uint8_t * smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t * full_k = reinterpret_cast<uint64_t *>(smem + L::kBars);
    uint64_t * full_v = full_k + L::kStages;
    uint64_t * empty = full_v + L::kStages;
    volatile int * flags = reinterpret_cast<volatile int *>(smem + L::kFlags);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(full_k + i, 1);
            mbar_init(full_v + i, 1);
            mbar_init(empty + i, kConsumers);
        }
        flags[0] = 0;
        mbar_init_fence();
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    const View & v = p.view;
    Walk * walks = reinterpret_cast<Walk *>(smem + L::kWalk);
    if (!walk_begin<kItemRows>(v, reinterpret_cast<uint64_t *>(smem), walks)) return;
    Walk & w = walks[warp];

    if (warp >= kConsumers) {
        const bool is_v = warp > kConsumers;
        const CUtensorMap * map = is_v ? &map_v : &map_k;
        uint64_t * full = is_v ? full_v : full_k;
        uint32_t n = 0;
        bool ok = true;
        do {
            uint32_t t0, t1;
            walk_segment<kItemRows>(w, t0, t1);
            const int32_t * row = v.table + uint64_t(w.b) * v.table_stride;
            const uint32_t begin = w.k.begin, hi = w.k.hi, head = w.kv_head;
            auto pages_of = [&](uint32_t t) {
                const uint32_t key0 = begin + t * kTileKeys;
                return tile_pages(v, row, key0, hi <= key0 ? key0 : min(hi, key0 + uint32_t(kTileKeys)));
            };
            TileLoad next = pages_of(t0);
            for (uint32_t t = t0; t < t1; ++t, ++n) {
                const TileLoad load = next;
                if (t + 1 < t1) next = pages_of(t + 1);
                const uint32_t st = n % L::kStages, turn = n / L::kStages;
                if (turn > 0) ok = __all_sync(0xffffffffu, mbar_wait(empty + st, (turn - 1) & 1, flags, v.error));
                if (!ok) break;
                tile_issue<D>(load, map, head, smem_u32(smem) + st * L::kStage + (is_v ? kTileBytes<D> : 0u), full + st);
            }
        } while (ok && walk_warp_next<kItemRows>(v, &w));
        if (flags[0]) {
            for (uint32_t i = n > uint32_t(L::kStages) ? n - L::kStages : 0u; i < n; ++i) {
                mbar_drain(full + i % L::kStages, (i / L::kStages) & 1);
            }
        }
        return;
    }

    // consumers
    const uint32_t grp = lane >> 2, tig = lane & 3;
    const uint32_t G = v.group, hd = v.head_dim;
    const float scale2 = p.scale * kLog2e;
    float * merge = reinterpret_cast<float *>(smem + L::kMerge);
    float2 * ml = reinterpret_cast<float2 *>(smem + L::kMl);
    uint32_t n = 0;
    do {
        uint32_t t0, t1;
        walk_segment<kItemRows>(w, t0, t1);
        const uint32_t packed = w.s.count * G;  // rows of an item: below 2^32 (checked on the host)
        const uint32_t row0 = w.tile * kRowsM;
        const int64_t first = int64_t(w.s.kv) - w.s.count;
        // Q fragments of rows grp and grp + 8
        uint32_t qa[D / 16][4];
        int32_t pos[2];
        uint32_t token_row[2], head[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t r = row0 + grp + 8 * e;
            const bool valid = r < packed;
            const uint32_t i = valid ? r / G : 0u, g = valid ? r % G : 0u;
            token_row[e] = w.s.q0 + i;
            head[e] = w.kv_head * G + g;
            pos[e] = int32_t(first + i);
            const T * src = static_cast<const T *>(p.q) + uint64_t(token_row[e]) * p.q_stride + uint64_t(head[e]) * hd;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t d = kk * 16 + h * 8;
                    qa[kk][e + 2 * h] = valid && d < hd ? *reinterpret_cast<const uint32_t *>(src + d + tig * 2) : 0u;
                }
            }
        }
        const int32_t pos_first = int32_t(first + row0 / G);
        const int32_t pos_last = int32_t(first + (min(row0 + uint32_t(kRowsM), packed) - 1) / G);
        float o[D / 8][4];
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        for (uint32_t t = t0; t < t1; ++t, ++n) {
            const uint32_t st = n % L::kStages, parity = (n / L::kStages) & 1;
            const uint32_t kbase = smem_u32(smem) + st * L::kStage, vbase = kbase + kTileBytes<D>;
            const int32_t key = int32_t(w.k.begin + t * kTileKeys + warp * 16);  // this warp's first key
            // after a wait that gave up the tiles are skipped, but every warp
            // still meets the others at the segments' barriers
            if (__any_sync(0xffffffffu, flags[0]) || !__all_sync(0xffffffffu, mbar_wait(full_k + st, parity, flags, v.error))) continue;
            float s[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
            }
            const uint32_t krow = warp * 16 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                uint32_t b[4];
                const uint32_t chunk = kk * 2 + ((lane >> 3) & 1);
                ldsm4(b, kbase + (chunk >> 3) * (kTileKeys * 128) + krow * 128 + (((chunk & 7) ^ (krow & 7)) << 4));
                mma_16816<T>(s[0], qa[kk], b[0], b[1]);
                mma_16816<T>(s[1], qa[kk], b[2], b[3]);
            }
            if (key + 15 > pos_first || (v.window > 0 && key <= pos_last - int32_t(v.window))) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int32_t k = key + j * 8 + int32_t(tig) * 2 + (e & 1), q = pos[e >> 1];
                        if (k > q || (v.window > 0 && k <= q - int32_t(v.window))) s[j][e] = -INFINITY;
                    }
                }
            }
            float alpha[2];
            uint32_t pa[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float mx = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                mx = fmaxf(m[e], mx * scale2);
                const float base = mx == -INFINITY ? 0.0f : mx;  // nothing seen yet: every term is 0
                alpha[e] = exp2_approx(m[e] - base);
                m[e] = mx;
                float q[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) q[c] = exp2_approx(fmaf(s[c >> 1][2 * e + (c & 1)], scale2, -base));
                l[e] = l[e] * alpha[e] + ((q[0] + q[1]) + (q[2] + q[3]));
                pa[e] = Num<T>::pack(q[0], q[1]);
                pa[e + 2] = Num<T>::pack(q[2], q[3]);
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    o[j][0] *= alpha[0];
                    o[j][1] *= alpha[0];
                    o[j][2] *= alpha[1];
                    o[j][3] *= alpha[1];
                }
            }
            if (!__all_sync(0xffffffffu, mbar_wait(full_v + st, parity, flags, v.error))) continue;
            // what no row sees may hold anything: its probability is 0, but 0 x NaN is not
            const bool clean = key < int32_t(w.k.lo) || key + 16 > int32_t(w.k.hi);
            if (clean) {
                for (int r = 0; r < 16; ++r) {
                    if (key + r >= int32_t(w.k.lo) && key + r < int32_t(w.k.hi)) continue;
                    for (uint32_t c = lane; c < D / 8; c += 32) {
                        const uint32_t at = vbase + (c >> 3) * (kTileKeys * 128) + (warp * 16 + r) * 128 + ((c & 7) << 4);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                    }
                }
                __syncwarp();
            }
            const uint32_t vrow = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
            for (int j = 0; j < D / 8; j += 2) {
                uint32_t b[4];
                const uint32_t chunk = j + (lane >> 4);
                ldsm4_trans(b, vbase + (chunk >> 3) * (kTileKeys * 128) + vrow * 128 + (((chunk & 7) ^ (vrow & 7)) << 4));
                mma_16816<T>(o[j], pa, b[0], b[1]);
                mma_16816<T>(o[j + 1], pa, b[2], b[3]);
            }
            if (clean) fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + st);
        }

        // the warps' parts of the segment
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
            if (tig == 0) ml[warp * kRowsM + grp + 8 * e] = make_float2(m[e], l[e]);
        }
        bar_consumers();
        float part[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float top = -INFINITY;
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) top = fmaxf(top, ml[x * kRowsM + grp + 8 * e].x);
            part[e] = m[e] == -INFINITY ? 0.0f : exp2_approx(m[e] - top);
        }
        const uint32_t orow = threadIdx.x >> 4, oc = (threadIdx.x & 15) * 4;  // output row and columns of this thread
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int x = 0; x < kConsumers; ++x) top = fmaxf(top, ml[x * kRowsM + orow].x);
#pragma unroll
        for (int x = 0; x < kConsumers; ++x) {
            const float2 a = ml[x * kRowsM + orow];
            sum += a.x == -INFINITY ? 0.0f : a.y * exp2_approx(a.x - top);
        }
        const uint32_t r = row0 + orow;
        const RowsOut<T> out(p, r < packed, w.s.q0 + r / G, w.kv_head * G + r % G);
        const bool whole = t0 == 0 && t1 == w.k.tiles;
        float * slot = p.partial + uint64_t(2 * blockIdx.x + (t0 == 0 ? 1 : 0)) * kSlotFloats;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t c = j * 8 + tig * 2;
                float * a = merge + (warp * kRowsM + grp) * 64 + (c ^ ((grp & 3) << 3));
                *reinterpret_cast<float2 *>(a) = make_float2(o[h * 8 + j][0] * part[0], o[h * 8 + j][1] * part[0]);
                *reinterpret_cast<float2 *>(a + 8 * 64) = make_float2(o[h * 8 + j][2] * part[1], o[h * 8 + j][3] * part[1]);
            }
            bar_consumers();
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) {
                const float4 a = *reinterpret_cast<const float4 *>(merge + (x * kRowsM + orow) * 64 + (oc ^ ((orow & 3) << 3)));
                acc.x += a.x;
                acc.y += a.y;
                acc.z += a.z;
                acc.w += a.w;
            }
            if (whole) out.store4(h * 64 + oc, acc, sum, hd);
            else __stcg(reinterpret_cast<float4 *>(slot + orow * D + h * 64 + oc), acc);
            bar_consumers();
        }
        if (whole) {
            if ((threadIdx.x & 15) == 0) out.store_lse(p, top, sum);
        } else {
            if ((threadIdx.x & 15) == 0) __stcg(reinterpret_cast<float2 *>(slot + kRowsM * D + 2 * orow), make_float2(top, sum));
            // the last CTA of the item to arrive joins the parts, in CTA order
            uint32_t c0, c1;
            walk_owners<kItemRows>(w, c0, c1);
            __threadfence();
            bar_consumers();
            if (threadIdx.x == 0) {
                const bool last = atomicAdd(p.counters + c0, 1u) == c1 - c0;
                if (last) p.counters[c0] = 0;
                flags[1] = last;
            }
            bar_consumers();
            if (flags[1]) {
                __threadfence();
                auto part_of = [&](uint32_t c) { return p.partial + uint64_t(2 * c + (c == c0 ? 1 : 0)) * kSlotFloats; };
                float jtop = -INFINITY;
                for (uint32_t c = c0; c <= c1; ++c) jtop = fmaxf(jtop, __ldcg(part_of(c) + kRowsM * D + 2 * orow));
                float jsum = 0.0f;
                float4 acc[D / 64];
#pragma unroll
                for (int h = 0; h < D / 64; ++h) acc[h] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                for (uint32_t c = c0; c <= c1; ++c) {
                    const float * from = part_of(c);
                    const float2 a = __ldcg(reinterpret_cast<const float2 *>(from + kRowsM * D + 2 * orow));
                    const float f = a.x == -INFINITY ? 0.0f : exp2_approx(a.x - jtop);
                    jsum = fmaf(a.y, f, jsum);
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) {
                        const float4 x = __ldcg(reinterpret_cast<const float4 *>(from + orow * D + h * 64 + oc));
                        acc[h].x = fmaf(x.x, f, acc[h].x);
                        acc[h].y = fmaf(x.y, f, acc[h].y);
                        acc[h].z = fmaf(x.z, f, acc[h].z);
                        acc[h].w = fmaf(x.w, f, acc[h].w);
                    }
                }
#pragma unroll
                for (int h = 0; h < D / 64; ++h) out.store4(h * 64 + oc, acc[h], jsum, hd);
                if ((threadIdx.x & 15) == 0) out.store_lse(p, jtop, jsum);
            }
            bar_consumers();
        }
    } while (walk_warp_next<kItemRows>(v, &w));
}

template <typename T, int D>
jfb_status launch_rows(const CUtensorMap & k, const CUtensorMap & v, const AttentionParams & p, const Device & device,
                       cudaStream_t s) {
    cudaError_t e = allow_smem<paged_rows_kernel<T, D>>(device, RowsSmem<D>::kBytes);
    if (e == cudaSuccess) e = launch_k(paged_rows_kernel<T, D>, dim3(device.sms), dim3(kThreadsRows), RowsSmem<D>::kBytes, s, k, v, p);
    if (e != cudaSuccess) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention: %s", cudaGetErrorString(e));
    return launch_status("jfb_paged_attention");
}

}  // namespace
}  // namespace paged
}  // namespace jfb

using namespace jfb;
using namespace jfb::paged;

extern "C" uint64_t jfb_paged_attention_workspace_bytes(void) {
    return kCounterBytes + uint64_t(current_device().sms) * 2 * kSlotFloats * sizeof(float);
}

extern "C" jfb_status jfb_paged_attention(const void * q, uint64_t q_stride, uint32_t rows, uint32_t heads, float scale,
                                          uint32_t window, const jfb_paged_cache * cache, const jfb_paged_batch * batch,
                                          void * out, uint64_t out_stride, float * lse, void * workspace,
                                          uint64_t workspace_bytes, int32_t * error_flag, void * stream) {
    jfb_status st = check_cache(cache);
    if (st.code == JFB_STATUS_OK) st = check_batch(batch, true);
    if (st.code == JFB_STATUS_OK) st = check_rows("jfb_paged_attention", q, q_stride, rows, heads, *cache);
    if (st.code == JFB_STATUS_OK) st = check_rows("jfb_paged_attention", out, out_stride, rows, heads, *cache);
    if (st.code != JFB_STATUS_OK) return st;
    if (!(scale > 0.0f) || scale > 3.0e38f || window > 0x7fffffffu) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_attention needs a positive finite scale and a window below 2^31");
    }
    const Device device = current_device();
    const uint32_t sms = device.sms;
    if (sms == 0 || sms * 2 * sizeof(uint32_t) > kCounterBytes) {
        return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention: no usable device");
    }
    const uint64_t need = kCounterBytes + uint64_t(sms) * 2 * kSlotFloats * sizeof(float);
    if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_attention needs a 16-byte aligned workspace of %llu bytes",
                            static_cast<unsigned long long>(need));
    }
    if (rows == 0 || batch->sequences == 0) return status_ok();
    AttentionParams p;
    p.view = make_view(*cache, *batch, rows, heads / cache->kv_heads, window, error_flag);
    p.view.item_rows = kRowsM;
    p.q = q;
    p.out = out;
    p.lse = lse;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.heads = heads;
    p.scale = scale;
    p.counters = static_cast<uint32_t *>(workspace);
    p.partial = reinterpret_cast<float *>(static_cast<uint8_t *>(workspace) + kCounterBytes);
    CUtensorMap mk, mv;
    if (!pool_map(mk, cache->k, *cache) || !pool_map(mv, cache->v, *cache)) {
        return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention: could not encode a TMA tensor map");
    }
    cudaStream_t s = as_stream(stream);
    const bool half = cache->dtype == JFB_DTYPE_F16;
    const uint32_t group = p.view.group;
    if (group <= 128 && uint64_t(rows) * group > 32ull * batch->sequences) return launch_attention_tc(*cache, mk, mv, p, device, s);
    if (cache->head_dim <= 64) {
        return half ? launch_rows<__half, 64>(mk, mv, p, device, s) : launch_rows<__nv_bfloat16, 64>(mk, mv, p, device, s);
    }
    return half ? launch_rows<__half, 128>(mk, mv, p, device, s) : launch_rows<__nv_bfloat16, 128>(mk, mv, p, device, s);
}
