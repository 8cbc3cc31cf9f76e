// Attention of chunks over a cache in pages on the tcgen05 tensor cores.
//
// An item is 256 packed rows (token, head of the group) of one sequence and kv
// head, two tiles of 128, and its keys come in tiles of 128. One CTA per SM
// walks its share of the units (walk_begin):
//   warps 0-3, 4-7  softmax of row tile 0 and 1, a thread per row: scores from
//                   tensor memory, running maximum and sum, probabilities back
//                   over the scores as the 16-bit A operand, results out;
//   warp 8          MMA: S_x = Q_x K^T and O_x += P_x V, so that one row tile's
//                   products run under the other's softmax;
//   warps 9, 10     K and V tiles, page by page through TMA, into one ring.
// Tensor memory (512 columns): S_0, S_1, O_0, O_1 of 128 f32 columns; P_x
// takes the first 64 columns of S_x. An MMA chain executes in issue order, so
// S_x of the next tile is issued right behind the P_x V that still reads P_x.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 over the
// one its sums refer to (the sums stay far inside f32's range and the
// probabilities below 2^8 keep their relative precision), so most tiles touch
// O not at all.
#include "paged_attention.cuh"
#include "paged_tc.cuh"

namespace jfb {
namespace paged {
namespace {

constexpr int kRowsTc = 256;
constexpr int kThreadsTc = 384;
constexpr int kMmaWarp = 8, kWarpK = 9, kWarpV = 10;
constexpr uint32_t kColS = 0, kColO = 256;  // of row tile 0; tile 1 is 128 columns further
constexpr float kSlack = 8.0f;              // growth of the maximum (log 2) that a rescale waits for

template <int D>
struct TcSmem {
    static constexpr int kStages = D == 128 ? 5 : 10;
    static constexpr uint32_t kQ = 2 * 128 * D * 2;
    static constexpr uint32_t kBars = kQ + kStages * kTileBytes<D>;
    static constexpr uint32_t kNumBars = 2 * kStages + 8;  // full, empty; s, p, o, q of both row tiles
    static constexpr uint32_t kWalk = kBars + kNumBars * 8;
    static constexpr uint32_t kFlags = kWalk + (sizeof(Walk) + 15) / 16 * 16;  // abort, last of tile 0 and 1, tmem
    static constexpr uint32_t kBytes = kFlags + 32 + 1024;
};
static_assert(TcSmem<128>::kBytes <= 232448 && TcSmem<64>::kBytes <= 232448);
static_assert(TcSmem<64>::kBars >= JFB_PAGED_MAX_SEQUENCES * 8);

template <typename T>
__device__ __forceinline__ const T * query_row(const AttentionParams & p, const Walk & w, uint32_t r) {
    if (r >= w.s.count * p.group) return nullptr;
    return static_cast<const T *>(p.q) + uint64_t(w.s.q0 + r / p.group) * p.q_stride +
           uint64_t(w.kv_head * p.group + r % p.group) * p.view.head_dim;
}

__device__ __forceinline__ bool two_tiles(const AttentionParams & p, const Walk & w) {
    return w.s.count * p.group > w.tile * kRowsTc + 128;
}

// The 128 threads of one row tile's softmax.
__device__ __forceinline__ void bar_tile(uint32_t x) {
    if (x == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
    else asm volatile("bar.sync 2, 128;" ::: "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreadsTc, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttentionParams p) {
    extern __shared__ uint8_t smem_raw[];
    using L = TcSmem<D>;
    uint8_t * smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint64_t * full = reinterpret_cast<uint64_t *>(smem + L::kBars);
    uint64_t * empty = full + L::kStages;
    uint64_t * s_full = empty + L::kStages;
    uint64_t * p_full = s_full + 2;
    uint64_t * o_full = p_full + 2;
    uint64_t * q_full = o_full + 2;
    volatile int * flags = reinterpret_cast<volatile int *>(smem + L::kFlags);
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(smem + L::kFlags + 16);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(s_full + x, 1);
            mbar_init(p_full + x, 4);
            mbar_init(o_full + x, 1);
            mbar_init(q_full + x, 4);
        }
        flags[0] = 0;
        mbar_init_fence();
    }
    pdl_trigger();
    pdl_wait();
    const View & v = p.view;
    Walk w;
    if (!walk_begin<kRowsTc>(v, p.group, p.window, reinterpret_cast<uint64_t *>(smem), reinterpret_cast<Walk *>(smem + L::kWalk), w)) {
        return;
    }
    fence_proxy_async();  // the ring held the walk's scratch
    if (warp == kMmaWarp) tmem_alloc(tmem_slot);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t ring = smem_u32(smem) + L::kQ;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == kWarpK || warp == kWarpV) {
            const bool is_v = warp == kWarpV;
            const CUtensorMap * map = is_v ? &map_v : &map_k;
            uint32_t n = is_v ? 1 : 0;  // ring slots alternate K, V
            bool ok = true;
            do {
                uint32_t t0, t1;
                walk_segment(w, t0, t1);
                const int32_t * row = v.table + uint64_t(w.b) * v.table_stride;
                for (uint32_t t = t0; t < t1; ++t, n += 2) {
                    const uint32_t st = n % L::kStages, turn = n / L::kStages;
                    if (turn > 0) ok = __all_sync(0xffffffffu, mbar_wait(empty + st, (turn - 1) & 1, flags, v.error));
                    if (!ok) break;
                    const uint32_t key0 = w.k.begin + t * kTileKeys;
                    const uint32_t key1 = w.k.hi <= key0 ? key0 : min(w.k.hi, key0 + uint32_t(kTileKeys));
                    load_tile<D>(v, map, row, w.kv_head, key0, key1, ring + st * kTileBytes<D>, full + st);
                }
            } while (ok && walk_next<kRowsTc>(v, p.group, p.window, w));
            if (flags[0]) {
                for (uint32_t i = n >= 2u * L::kStages ? n - 2u * L::kStages : (is_v ? 1u : 0u); i < n; i += 2) {
                    mbar_drain(full + i % L::kStages, (i / L::kStages) & 1);
                }
            }
        } else if (warp == kMmaWarp) {
            constexpr uint32_t idesc_s = instr_desc<T>(kTileKeys, false), idesc_o = instr_desc<T>(D, true);
            const uint32_t q_addr = smem_u32(smem);
            uint32_t tiles[2] = {0, 0}, items[2] = {0, 0};
            uint32_t g = 0;  // key tiles so far
            bool ok = true;
            auto wait = [&](uint64_t * bar, uint32_t parity) {
                ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, flags, v.error));
                return ok;
            };
            auto full_of = [&](uint32_t n) { return wait(full + n % L::kStages, (n / L::kStages) & 1); };
            auto issue_s = [&](uint32_t x, uint32_t n) {
                const uint32_t k_addr = ring + (n % L::kStages) * kTileBytes<D>;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t at = (kk >> 2) * kHalfBytes + (kk & 3) * 32;
                    mma_ss(tmem + kColS + x * 128, desc_k_major(q_addr + x * (128 * D * 2) + at), desc_k_major(k_addr + at), idesc_s, kk > 0);
                }
                mma_commit(s_full + x);
            };
            do {
                uint32_t t0, t1;
                walk_segment(w, t0, t1);
                const uint32_t last = two_tiles(p, w) ? 1 : 0;
                if (!full_of(2 * g)) break;
                for (uint32_t x = 0; x <= last; ++x) {
                    if (!wait(q_full + x, items[x]++ & 1)) break;
                    tc_fence_after();
                    issue_s(x, 2 * g);
                }
                if (!ok) break;
                mma_commit(empty + (2 * g) % L::kStages);
                for (uint32_t t = t0; ok && t < t1; ++t, ++g) {
                    const uint32_t vs = (2 * g + 1) % L::kStages;
                    const uint32_t v_addr = ring + vs * kTileBytes<D>;
                    for (uint32_t x = 0; x <= last; ++x) {
                        if (!wait(p_full + x, tiles[x]++ & 1)) break;
                        if (x == 0) {
                            if (!full_of(2 * g + 1)) break;
                            // what no row sees may hold anything: its probability is 0, but 0 x NaN is not
                            const uint32_t key0 = w.k.begin + t * kTileKeys;
                            if (key0 < w.k.lo || key0 + kTileKeys > w.k.hi) {
                                for (uint32_t r = 0; r < uint32_t(kTileKeys); ++r) {
                                    if (key0 + r >= w.k.lo && key0 + r < w.k.hi) continue;
                                    if (lane < D / 8) {
                                        const uint32_t at = v_addr + (lane >> 3) * kHalfBytes + r * 128 + ((lane & 7) << 4);
                                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                                    }
                                }
                                fence_proxy_async();
                                __syncwarp();
                            }
                        }
                        tc_fence_after();
#pragma unroll
                        for (int kk = 0; kk < kTileKeys / 16; ++kk) {
                            mma_ts(tmem + kColO + x * 128, tmem + kColS + x * 128 + kk * 8, desc_mn_major(v_addr + kk * 2048), idesc_o,
                                   t > t0 || kk > 0);
                        }
                        mma_commit(o_full + x);
                        if (x == last) mma_commit(empty + vs);
                        if (t + 1 < t1) {
                            if (x == 0 && !full_of(2 * g + 2)) break;
                            issue_s(x, 2 * g + 2);
                            if (x == last) mma_commit(empty + (2 * g + 2) % L::kStages);
                        }
                    }
                }
            } while (ok && walk_next<kRowsTc>(v, p.group, p.window, w));
            if (flags[0]) {  // MMAs in flight finish before tensor memory is given back
                const uint64_t t = global_ns();
                mma_commit(q_full);
                while (global_ns() - t < 10000000ull) __nanosleep(1000);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const uint32_t x = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = tmem + ((warp & 3) << 21);  // this warp's 32 lanes
        const uint32_t t_s = lanes + kColS + x * 128, t_o = lanes + kColO + x * 128;
        const float scale2 = p.scale * kLog2e;
        uint32_t n = 0;  // tiles of this row tile so far
        auto load_q = [&]() {
            store_row<T, D>(smem + x * (128 * D * 2), row, query_row<T>(p, w, w.tile * kRowsTc + x * 128 + row), v.head_dim);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + x);
        };
        bool more = true;
        while (more && x == 1 && !two_tiles(p, w)) more = walk_next<kRowsTc>(v, p.group, p.window, w);
        if (more) load_q();
        while (more) {
            uint32_t t0, t1;
            walk_segment(w, t0, t1);
            const uint32_t packed = w.s.count * p.group, r0 = w.tile * kRowsTc + x * 128;
            const int64_t first = int64_t(w.s.kv) - w.s.count;
            const int32_t pos = int32_t(first + (r0 + row) / p.group);
            const int32_t pos_first = int32_t(first + r0 / p.group);
            const int32_t pos_last = int32_t(first + (min(r0 + 128, packed) - 1) / p.group);
            float m = -INFINITY, l0 = 0.0f, l1 = 0.0f;
            for (uint32_t t = t0; t < t1; ++t, ++n) {
                // after a wait that gave up the tiles are skipped; the warps still meet at the barriers below
                if (__any_sync(0xffffffffu, flags[0]) || !__all_sync(0xffffffffu, mbar_wait(s_full + x, n & 1, flags, v.error))) continue;
                tc_fence_after();
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, s + c * 32);
                tmem_wait_ld();
                const int32_t key0 = int32_t(w.k.begin + t * kTileKeys);
                if (key0 + kTileKeys - 1 > pos_first || (p.window > 0 && key0 <= pos_last - int32_t(p.window))) {
                    const int32_t hi = pos - key0, lo = p.window > 0 ? hi - int32_t(p.window) : -1;
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = i <= hi && i > lo ? s[i] : -INFINITY;
                }
                float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < 128; i += 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[i + e]);
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
                const bool grow = top > m + kSlack;
                if (__any_sync(0xffffffffu, grow)) {
                    const float next = grow ? top : m;
                    const float f = grow ? exp2_approx(m - next) : 1.0f;
                    m = next;
                    l0 *= f;
                    l1 *= f;
                    if (t > t0) {
                        if (!__all_sync(0xffffffffu, mbar_wait(o_full + x, (n - 1) & 1, flags, v.error))) continue;
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            float o[32];
                            tmem_ld32(t_o + c * 32, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= f;
                            tmem_st32(t_o + c * 32, reinterpret_cast<const uint32_t *>(o));
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.0f : -m;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        float a, b;
                        fma2(a, b, s[c * 32 + i], s[c * 32 + i + 1], scale2, base);
                        a = exp2_approx(a);
                        b = exp2_approx(b);
                        add2(l0, l1, a, b);
                        pk[i / 2] = Num<T>::pack(a, b);
                    }
                    tmem_st16(t_s + c * 16, pk);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + x);
            }
            // the segment's results; the next item's rows are fetched first, so its products can start
            const RowsOut<T> out(p, w, r0 + row);
            const bool whole = t0 == 0 && t1 == w.k.units;
            const uint32_t c0 = cta_of(w.item0, w.total, w.ctas), c1 = cta_of(w.item0 + w.k.units - 1, w.total, w.ctas);
            do {
                more = walk_next<kRowsTc>(v, p.group, p.window, w);
            } while (more && x == 1 && !two_tiles(p, w));
            if (more) load_q();
            const bool ok = __all_sync(0xffffffffu, flags[0] == 0 && mbar_wait(o_full + x, (n - 1) & 1, flags, v.error));
            tc_fence_after();
            const float sum = l0 + l1;
            // parts are stored as [4 columns][row] so that a warp's stores are contiguous
            float * slot = p.partial + uint64_t(2 * blockIdx.x + (t0 == 0 ? 1 : 0)) * kSlotFloats;
            if (ok) {
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    float o[32];
                    tmem_ld32(t_o + c * 32, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 a = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        const uint32_t d = c * 32 + i;
                        if (whole) out.store4(d, a, sum, v.head_dim);
                        else __stcg(reinterpret_cast<float4 *>(slot) + (d / 4) * kRowsTc + x * 128 + row, a);
                    }
                }
                if (whole) out.store_lse(p, m, sum);
                else __stcg(reinterpret_cast<float2 *>(slot + kRowsTc * D) + x * 128 + row, make_float2(m, sum));
            }
            tc_fence_before();
            if (!whole) {
                // the last CTA of the item to arrive joins this row tile's parts, in CTA order
                __threadfence();
                bar_tile(x);
                if (row == 0) {
                    const bool last = atomicAdd(p.counters + 2 * c0 + x, 1u) == c1 - c0;
                    if (last) p.counters[2 * c0 + x] = 0;
                    flags[1 + x] = last;
                }
                bar_tile(x);
                if (flags[1 + x]) {
                    __threadfence();
                    auto part_of = [&](uint32_t c) { return p.partial + uint64_t(2 * c + (c == c0 ? 1 : 0)) * kSlotFloats; };
                    auto ml_of = [&](uint32_t c) { return __ldcg(reinterpret_cast<const float2 *>(part_of(c) + kRowsTc * D) + x * 128 + row); };
                    float jtop = -INFINITY, jsum = 0.0f;
                    for (uint32_t c = c0; c <= c1; ++c) jtop = fmaxf(jtop, ml_of(c).x);
                    for (uint32_t c = c0; c <= c1; ++c) {
                        const float2 a = ml_of(c);
                        jsum = fmaf(a.y, a.x == -INFINITY ? 0.0f : exp2_approx(a.x - jtop), jsum);
                    }
#pragma unroll
                    for (int d = 0; d < D; d += 32) {
                        float4 acc[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        for (uint32_t c = c0; c <= c1; ++c) {
                            const float a = ml_of(c).x;
                            const float f = a == -INFINITY ? 0.0f : exp2_approx(a - jtop);
                            const float4 * from = reinterpret_cast<const float4 *>(part_of(c)) + (d / 4) * kRowsTc + x * 128 + row;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float4 y = __ldcg(from + i * kRowsTc);
                                acc[i].x = fmaf(y.x, f, acc[i].x);
                                acc[i].y = fmaf(y.y, f, acc[i].y);
                                acc[i].z = fmaf(y.z, f, acc[i].z);
                                acc[i].w = fmaf(y.w, f, acc[i].w);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) out.store4(d + i * 4, acc[i], jsum, v.head_dim);
                    }
                    out.store_lse(p, jtop, jsum);
                }
                bar_tile(x);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) tmem_free(tmem);
}

template <typename T, int D>
jfb_status launch(const CUtensorMap & k, const CUtensorMap & v, const AttentionParams & p, uint32_t sms, cudaStream_t s) {
    auto kernel = paged_tc_kernel<T, D>;
    cudaError_t e = allow_smem(kernel, TcSmem<D>::kBytes);
    if (e == cudaSuccess) e = launch_k(kernel, dim3(sms), dim3(kThreadsTc), TcSmem<D>::kBytes, s, k, v, p);
    if (e != cudaSuccess) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention: %s", cudaGetErrorString(e));
    return launch_status("jfb_paged_attention");
}

}  // namespace

jfb_status launch_attention_tc(bool half, uint32_t head_dim, const CUtensorMap & k, const CUtensorMap & v, const AttentionParams & p,
                               uint32_t sms, cudaStream_t s) {
    if (head_dim <= 64) return half ? launch<__half, 64>(k, v, p, sms, s) : launch<__nv_bfloat16, 64>(k, v, p, sms, s);
    return half ? launch<__half, 128>(k, v, p, sms, s) : launch<__nv_bfloat16, 128>(k, v, p, sms, s);
}

}  // namespace paged
}  // namespace jfb
