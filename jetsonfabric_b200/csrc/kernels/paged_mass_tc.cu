// The attention weight each cached key received from chunks of new tokens, on
// the tcgen05 tensor cores.
//
// The keys are the M side, so that every sum over rows stays in one thread: an
// item is 256 keys of one sequence and kv head, two key tiles, its steps the
// row tiles (128 / G whole tokens) that see any of them, S^T = K Q^T of a step
// 2 x 128 x 128 scores. A step costs one exponential per score, 2048 cycles of
// the unit against 1024 of the tensor pipe and 32 KB of queries, so the
// exponentials bound the time (with 128 keys an item the queries' way from L2
// did: 250 us for chunks of 700 to 2048 tokens over 2048 to 8000 keys, 16/2 heads;
// 152 to 157 now). A cluster of 4 CTAs takes an item, every fourth
// step each, and adds the four sums over distributed shared memory: few long
// items still fill the SMs, and no workspace or order of arrival is involved.
// Where items are many or their steps few, the CTAs of a cluster take items of
// their own instead (items_apart; 64 sequences of 1150 keys with 8 new tokens,
// 28/4 heads: 83 us, 223 shared).
// Workers take whole items off the evenly divided line of units
// (walk_locate), each the items whose middle lies in its part.
//   warps 0-7, 8-15  sums of key tile 0 and 1, two threads per key, each half
//                    of a step's rows (one thread per key, 8 warps, left the
//                    exponentials' unit idle a quarter of the time: 197 us);
//   warp 16          the MMAs, up to two steps ahead (S takes all of the 512
//                    columns of tensor memory);
//   warp 17          K tiles and queries through TMA;
//   warp 18          each row's -lse and slot.
#include "paged_attention.cuh"
#include "paged_mass.cuh"
#include "paged_tc.cuh"

namespace jfb {
namespace paged {
namespace {

constexpr int kItemMass = 16; // units of an item's start and end
constexpr int kThreadsMass = 608;
constexpr int kWarpMma = 16, kWarpLoad = 17, kWarpLse = 18;
constexpr uint32_t kCluster = 4;
constexpr uint32_t kItemKeys = 2 * kTileKeys;
constexpr uint32_t kLseRing = 8;  // steps of row data ahead

// Items of a sequence: its pairs of key tiles with the row tiles that see them.
struct KeyItems {
    struct Part {
        uint32_t first, tiles;  // row tiles [first, first + tiles)
    };
    static __device__ __forceinline__ uint32_t limit(const View & v, const Sequence & s) {
        if (s.kv <= v.slots) return s.kv;
        flag_error(v.error, JFB_PAGED_ERROR_RANGE);
        return uint32_t(v.slots);
    }
    static __device__ __forceinline__ uint32_t count(const View & v, const Sequence & s) {
        return (limit(v, s) + kItemKeys - 1) / kItemKeys;
    }
    static __device__ __forceinline__ Part part(const View & v, const Sequence & s, uint32_t item) {
        const uint32_t tokens = v.item_rows / v.group;
        const int64_t first = int64_t(s.kv) - s.count, key0 = int64_t(item) * kItemKeys;
        const int64_t key1 = key0 + kItemKeys < limit(v, s) ? key0 + kItemKeys : limit(v, s);
        const int64_t i0 = key0 > first ? key0 - first : 0;  // tokens [i0, i1) see some key of the tile
        int64_t i1 = s.count;
        if (v.window > 0 && key1 - 1 + v.window - first < i1) i1 = key1 - 1 + v.window - first;
        Part p = {0, 0};
        if (i0 < i1) {
            p.first = uint32_t(i0) / tokens;
            p.tiles = (uint32_t(i1) + tokens - 1) / tokens - p.first;
        }
        return p;
    }
};
using KeyTileWalk = WalkOf<KeyItems>;

template <int D>
struct MassTcSmem {
    static constexpr uint32_t kQStages = D == 128 ? 4 : 8;
    static constexpr uint32_t kQ = 2 * kTileBytes<D>;  // the two K tiles first
    static constexpr uint32_t kRows = kQ + kQStages * kTileBytes<D>;  // [ring][128] (-lse log2 e, slot)
    static constexpr uint32_t kSums = kRows + kLseRing * 128 * 8;     // [key tile][2][cluster][128]
    static constexpr uint32_t kHalves = kSums + 2 * 2 * kCluster * 128 * 4;  // [key tile][2][128] of the second threads
    static constexpr uint32_t kBars = kHalves + 2 * 2 * 128 * 4;
    static constexpr uint32_t kNumBars = 2 + 2 * kQStages + 8 + 2 * kLseRing + 8;
    static constexpr uint32_t kWalk = kBars + kNumBars * 8;
    static constexpr uint32_t kFlags = kWalk + kThreadsMass / 32 * sizeof(KeyTileWalk);  // abort, tmem
    static constexpr uint32_t kBytes = kFlags + 32;
};
static_assert(MassTcSmem<128>::kBytes <= 232448 && MassTcSmem<64>::kBytes <= 232448);
static_assert(MassTcSmem<64>::kBars >= JFB_PAGED_MAX_SEQUENCES * 8);

struct MassMaps {
    CUtensorMap k, q;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Shared-memory address of `p` in the CTA of cluster rank `rank`.
__device__ __forceinline__ uint32_t remote(const void * p, uint32_t rank) {
    uint32_t out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(smem_u32(p)), "r"(rank));
    return out;
}
__device__ __forceinline__ void remote_store(const float * p, uint32_t rank, float x) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote(p, rank)), "f"(x) : "memory");
}
// Releases the calling thread's (and, after a warp barrier and fence, its warp's) accesses.
__device__ __forceinline__ void remote_arrive(uint64_t * bar, uint32_t rank) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote(bar, rank)) : "memory");
}
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t * bar, uint32_t parity, volatile int * abort_flag, int32_t * error) {
    const uint64_t t0 = global_ns();
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.b32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(kSuspendNs)
            : "memory");
        if (ok != 0) return true;
        if (*abort_flag) return false;
        if (global_ns() - t0 > kWaitNs) break;
    }
    *abort_flag = 1;
    flag_error(error, JFB_PAGED_ERROR_TIMEOUT);
    return false;
}

// The next item, if its middle lies in the cluster's part of the line.
__device__ __forceinline__ bool step_item(const View & v, KeyTileWalk & w) {
    if (w.item0 + w.k.tiles + kItemMass >= w.end) return false;
    walk_item<kItemMass>(v, w);
    return w.item0 + (w.k.tiles + kItemMass) / 2 < w.end;
}
__device__ __forceinline__ bool next_item(const View & v, KeyTileWalk * w) {
    __syncwarp();
    int more = 0;
    if ((threadIdx.x & 31) == 0) more = step_item(v, *w);
    return __shfl_sync(0xffffffffu, more, 0) != 0;
}
// Whether the CTAs of a cluster take items of their own: where that makes the
// busiest one's time, counted in steps and 4 for an item's start and end (the
// longest item and as many mean ones as come before it), smaller than sharing
// each item's steps. Many sequences have many items.
__device__ __forceinline__ bool items_apart(const View & v, uint32_t ctas) {
    if (v.sequences > 128) return true;
    const uint32_t lane = threadIdx.x & 31, tokens = v.item_rows / v.group;
    float items = 0.0f, steps = 0.0f, most = 0.0f;
    for (uint32_t b = lane; b < v.sequences; b += 32) {
        const Sequence s = load_sequence(v, b);
        const float n = float(KeyItems::count(v, s)), of = float((s.count + tokens - 1) / tokens);
        items += n;
        steps += n * of;
        most = fmaxf(most, of);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        items += __shfl_xor_sync(0xffffffffu, items, d);
        steps += __shfl_xor_sync(0xffffffffu, steps, d);
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    }
    const float mean = steps / fmaxf(items, 1.0f), all = items * float(v.kv_heads);
    const auto time = [&](float workers, float sharing) {
        return fmaxf(ceilf(all / workers) - 1.0f, 0.0f) * (4.0f + ceilf(mean / sharing)) + 4.0f + ceilf(most / sharing);
    };
    return time(float(ctas), 1.0f) < time(float(ctas / kCluster), float(kCluster));
}
// Whether the item has keys in its second tile.
__device__ __forceinline__ bool two_key_tiles(const View & v, const KeyTileWalk & w) {
    return KeyItems::limit(v, w.s) > w.tile * kItemKeys + kTileKeys;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreadsMass, 1)
    mass_tc_kernel(const __grid_constant__ MassMaps maps, const MassParams p, const uint32_t tokens) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using L = MassTcSmem<D>;
    uint64_t * k_full = reinterpret_cast<uint64_t *>(smem + L::kBars);
    uint64_t * k_free = k_full + 1;
    uint64_t * q_full = k_free + 1;
    uint64_t * q_free = q_full + L::kQStages;
    uint64_t * s_full = q_free + L::kQStages;  // [key tile][2]
    uint64_t * s_free = s_full + 4;
    uint64_t * r_full = s_free + 4;
    uint64_t * r_free = r_full + kLseRing;
    uint64_t * sum_full = r_free + kLseRing;  // [key tile][2], of the leader: the cluster's sums of an even or odd item are in
    uint64_t * sum_free = sum_full + 4;       // of every CTA: the leader has used them
    volatile int * flags = reinterpret_cast<volatile int *>(smem + L::kFlags);
    uint32_t * tmem_slot = reinterpret_cast<uint32_t *>(smem + L::kFlags + 16);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = cluster_rank();
    if (threadIdx.x == 0) {
        mbar_init(k_full, 2);  // both key tiles
        mbar_init(k_free, 1);
        for (uint32_t i = 0; i < L::kQStages; ++i) {
            mbar_init(q_full + i, 1);
            mbar_init(q_free + i, 1);
        }
        for (uint32_t i = 0; i < 4; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(s_free + i, 8);
            mbar_init(sum_full + i, 4 * kCluster);
            mbar_init(sum_free + i, 1);
        }
        for (uint32_t i = 0; i < kLseRing; ++i) {
            mbar_init(r_full + i, 1);
            mbar_init(r_free + i, 16);
        }
        flags[0] = 0;
        mbar_init_fence();
    }
    pdl_trigger();
    pdl_wait();
    const View & v = p.view;
    KeyTileWalk * walks = reinterpret_cast<KeyTileWalk *>(smem + L::kWalk);
    const uint32_t share = items_apart(v, gridDim.x) ? 1u : kCluster, part = share == 1 ? 0u : rank;  // CTAs of an item
    walk_locate<kItemMass>(v, reinterpret_cast<uint64_t *>(smem), blockIdx.x / share, gridDim.x / share, walks);
    if (lane == 0) {
        KeyTileWalk & start = walks[warp];
        if (start.unit < start.end) {
            const uint64_t middle = start.item0 + (start.k.tiles + kItemMass) / 2;
            // an item whose middle lies before or behind this part is another cluster's
            if (middle >= start.end || (middle < start.unit && !step_item(v, start))) start.unit = start.end;
        }
    }
    __syncthreads();
    KeyTileWalk & w = walks[warp];
    const bool aligned = (smem_u32(smem) & 1023u) == 0;  // the swizzled tiles need it
    const bool work = w.unit < w.end && aligned;
    if (!aligned && threadIdx.x == 0) flag_error(v.error, JFB_PAGED_ERROR_TIMEOUT);
    // rows that no query fills stay zero (and this may have held the walk's scratch)
    for (uint32_t i = threadIdx.x; i < L::kRows / 16; i += kThreadsMass) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async();
    if (warp == kWarpMma) tmem_alloc(tmem_slot);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    cluster_sync();  // every CTA's barriers are initialised before any remote arrival
    const uint32_t tmem = *tmem_slot;
    bool ok = work;
    auto wait = [&](uint64_t * bar, uint32_t parity) {
        ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, flags, v.error));
        return ok;
    };
    // this CTA's steps of an item are row tiles k.first + part, + share, ...; s counts its steps over all items
    uint32_t s = 0;

    if (warp == kWarpLoad) {
        uint32_t item = 0;
        for (bool more = work; ok && more; ++item) {
            const uint32_t key0 = w.tile * kItemKeys, limit = KeyItems::limit(v, w.s);
            const int32_t * row = v.table + uint64_t(w.b) * v.table_stride;
            const TileLoad k0 = tile_pages(v, row, key0, min(limit, key0 + uint32_t(kTileKeys)));
            const uint32_t key1 = min(limit, key0 + uint32_t(kTileKeys));
            const TileLoad k1 = tile_pages(v, row, key1, min(limit, key0 + kItemKeys));
            if (item > 0 && !wait(k_free, (item - 1) & 1)) break;
            tile_issue<D>(v, k0, &maps.k, w.kv_head, smem_u32(smem), k_full);
            tile_issue<D>(v, k1, &maps.k, w.kv_head, smem_u32(smem) + kTileBytes<D>, k_full);
            for (uint32_t i = part; i < w.k.tiles; i += share, ++s) {
                const uint32_t st = s % L::kQStages;
                if (s >= L::kQStages && !wait(q_free + st, (s / L::kQStages - 1) & 1)) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(q_full + st, tokens * v.group * D * 2);
                    for (int h = 0; h < D / 64; ++h) {
                        tma_load_rows(smem_u32(smem) + L::kQ + st * kTileBytes<D> + h * kHalfBytes, &maps.q, h * 64,
                                      int32_t(w.kv_head * v.group), int32_t(w.s.q0 + (w.k.first + i) * tokens), q_full + st);
                    }
                }
                __syncwarp();
            }
            more = next_item(v, &w);
        }
        if (flags[0]) {
            if (item > 0) mbar_drain(k_full, (item - 1) & 1);
            for (uint32_t i = s >= L::kQStages ? s - L::kQStages : 0u; i < s; ++i) {
                mbar_drain(q_full + i % L::kQStages, (i / L::kQStages) & 1);
            }
        }
    } else if (warp == kWarpMma) {
        uint32_t item = 0, s1 = 0;  // steps of items with a second key tile
        for (bool more = work; ok && more; ++item) {
            const bool two = two_key_tiles(v, w);
            if (!wait(k_full, item & 1)) break;
            for (uint32_t i = part; i < w.k.tiles; i += share, ++s) {
                const uint32_t st = s % L::kQStages, q_addr = smem_u32(smem) + L::kQ + st * kTileBytes<D>;
                if (!wait(q_full + st, (s / L::kQStages) & 1)) break;
                for (uint32_t x = 0; x <= (two ? 1u : 0u); ++x) {
                    const uint32_t n = x == 0 ? s : s1++, buf = 2 * x + (n & 1);
                    if (n >= 2 && !wait(s_free + buf, (n / 2 - 1) & 1)) break;
                    tc_fence_after();
                    mma_scores<T, D>(tmem + buf * 128, smem_u32(smem) + x * kTileBytes<D>, q_addr);
                    mma_commit(s_full + buf);
                }
                mma_commit(q_free + st);
            }
            mma_commit(k_free);
            more = next_item(v, &w);
        }
        if (flags[0]) {  // MMAs in flight finish before tensor memory is given back
            const uint64_t t = global_ns();
            while (global_ns() - t < 10000000ull) __nanosleep(1000);
        }
    } else if (warp == kWarpLse) {
        float2 * ring = reinterpret_cast<float2 *>(smem + L::kRows);
        uint32_t token[4], head[4];  // of this lane's four rows
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            token[e] = (lane + 32 * e) / v.group;
            head[e] = lane + 32 * e - token[e] * v.group;
        }
        for (bool more = work; ok && more;) {
            const int64_t first = int64_t(w.s.kv) - w.s.count;
            for (uint32_t i = part; i < w.k.tiles; i += share, ++s) {
                const uint32_t st = s % kLseRing, token0 = (w.k.first + i) * tokens;
                float2 x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // rows of no token: weight 0, and before every slot
                    const bool valid = token[e] < tokens && token0 + token[e] < w.s.count;
                    x[e].x = valid ? -kLog2e * p.lse[uint64_t(w.s.q0 + token0 + token[e]) * p.heads + w.kv_head * v.group + head[e]] : -INFINITY;
                    x[e].y = __int_as_float(valid ? int32_t(first + token0 + token[e]) : -1);
                }
                if (s >= kLseRing && !wait(r_free + st, (s / kLseRing - 1) & 1)) break;
#pragma unroll
                for (int e = 0; e < 4; ++e) ring[st * 128 + lane + 32 * e] = x[e];
                __syncwarp();
                if (lane == 0) mbar_arrive(r_full + st);
            }
            more = next_item(v, &w);
        }
    } else if (warp < 16) {
        const uint32_t x = warp >> 3, half = (warp >> 2) & 1, key = threadIdx.x & 127;
        const uint32_t lanes = tmem + ((warp & 3) << 21);
        const float scale2 = p.scale * kLog2e;
        const float2 * ring = reinterpret_cast<const float2 *>(smem + L::kRows);
        float * sums = reinterpret_cast<float *>(smem + L::kSums) + x * 2 * kCluster * 128;
        float * halves = reinterpret_cast<float *>(smem + L::kHalves) + x * 256 + key;
        sum_full += 2 * x;
        sum_free += 2 * x;
        uint32_t item = 0, n = 0;  // items and steps of this key tile
        for (bool more = work; more;) {
            const int64_t first = int64_t(w.s.kv) - w.s.count;
            const uint32_t key0 = w.tile * kItemKeys + x * kTileKeys, at = key0 + key;
            const bool mine = x == 0 || two_key_tiles(v, w);
            const uint32_t first_tile = w.k.first, tiles = w.k.tiles, rows = w.s.count;
            // this thread's result, and what was there before: asked for now, like the next item, for their latency
            const bool writes = part == 0 && half == 0 && mine && at < KeyItems::limit(v, w.s);
            const uint64_t to = (uint64_t(w.b) * v.kv_heads + w.kv_head) * v.slots + at;
            const float before = writes && p.mass_in != nullptr && int64_t(at) < first ? p.mass_in[to] : 0.0f;
            more = next_item(v, &w);
            float total = 0.0f;
            for (uint32_t i = part; i < tiles; i += share, ++s) {
                const uint32_t st = s % kLseRing;
                // after a wait that gave up the steps are skipped; the warps still meet at the barriers below
                if (!wait(r_full + st, (s / kLseRing) & 1)) continue;
                if (mine) {
                    const uint32_t buf = 2 * x + (n & 1);
                    const uint32_t token0 = (first_tile + i) * tokens;
                    const int64_t pos0 = first + token0, pos1 = pos0 + tokens - 1;
                    const bool edge = token0 + tokens > rows || pos0 < int64_t(key0) + kTileKeys - 1 ||
                                      (v.window > 0 && int64_t(key0) <= pos1 - int64_t(v.window));
                    if (!wait(s_full + buf, (n / 2) & 1)) continue;
                    ++n;
                    tc_fence_after();
                    const float4 * data = reinterpret_cast<const float4 *>(ring + st * 128 + half * 64);
                    float a0 = 0.0f, a1 = 0.0f;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float y[32];
                        tmem_ld32(lanes + buf * 128 + half * 64 + c * 32, y);
                        tmem_wait_ld();
                        if (c == 1) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(s_free + buf);
                        }
                        if (edge) {
#pragma unroll
                            for (int j = 0; j < 32; j += 2) {
                                const float4 r = data[c * 16 + j / 2];
                                float e0, e1;
                                fma2(e0, e1, y[j], y[j + 1], scale2, r.x, r.z);
                                e0 = exp2_approx(e0);
                                e1 = exp2_approx(e1);
                                const int32_t p0 = __float_as_int(r.y), p1 = __float_as_int(r.w), k = int32_t(at);
                                e0 = k <= p0 && (v.window == 0 || k > p0 - int32_t(v.window)) ? e0 : 0.0f;
                                e1 = k <= p1 && (v.window == 0 || k > p1 - int32_t(v.window)) ? e1 : 0.0f;
                                add2(a0, a1, e0, e1);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; j += 2) {
                                const float4 r = data[c * 16 + j / 2];
                                float e0, e1;
                                fma2(e0, e1, y[j], y[j + 1], scale2, r.x, r.z);
                                add2(a0, a1, exp2_approx(e0), exp2_approx(e1));
                            }
                        }
                    }
                    total += a0 + a1;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(r_free + st);
            }
            if (mine) {  // the cluster's sums to the leader, which writes them
                const uint32_t q = item & 1, turn = item >> 1;
                ++item;
                if (half) halves[q * 128] = total;
                if (x == 0) asm volatile("bar.sync 1, 256;" ::: "memory");
                else asm volatile("bar.sync 2, 256;" ::: "memory");
                if (half) continue;
                total += halves[q * 128];
                if (share == 1) {
                    if (ok && writes) p.mass_out[to] = before + total;
                    continue;
                }
                if (turn > 0) ok = ok && __all_sync(0xffffffffu, mbar_wait_cluster(sum_free + q, (turn - 1) & 1, flags, v.error));
                if (ok) {
                    remote_store(sums + (q * kCluster + rank) * 128 + key, 0, total);
                    asm volatile("fence.acq_rel.cluster;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) remote_arrive(sum_full + q, 0);
                }
                if (rank == 0) {
                    ok = ok && __all_sync(0xffffffffu, mbar_wait_cluster(sum_full + q, turn & 1, flags, v.error));
                    if (ok && writes) {
                        float sum = 0.0f;
#pragma unroll
                        for (uint32_t r = 0; r < kCluster; ++r) sum += sums[(q * kCluster + r) * 128 + key];
                        p.mass_out[to] = before + sum;
                    }
                    if (x == 0) asm volatile("bar.sync 3, 128;" ::: "memory");
                    else asm volatile("bar.sync 4, 128;" ::: "memory");
                    if ((warp & 3) == 0 && lane < kCluster) remote_arrive(sum_free + q, lane);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kWarpMma) tmem_free(tmem);
    cluster_sync();  // no CTA leaves while another may still reach its shared memory
}

template <typename T, int D>
jfb_status launch(const MassMaps & maps, const MassParams & p, uint32_t tokens, const Device & device, cudaStream_t s) {
    constexpr auto kernel = mass_tc_kernel<T, D>;
    cudaError_t e = allow_smem<mass_tc_kernel<T, D>>(device, MassTcSmem<D>::kBytes);
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreadsMass);
    cfg.dynamicSmemBytes = MassTcSmem<D>::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    // as many clusters as the GPCs hold at once: the line is divided evenly among them
    const uint32_t most = device.sms / kCluster;
    cfg.gridDim = dim3(most * kCluster);
    static std::atomic<int> known[64];  // per device
    const bool keep = device.index >= 0 && device.index < 64;
    int n = keep ? known[device.index].load(std::memory_order_relaxed) : 0;
    if (e == cudaSuccess && n == 0) e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    if (e == cudaSuccess && (n < 1 || most < 1)) {
        return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention_mass: no room for a cluster");
    }
    if (e == cudaSuccess && keep) known[device.index].store(n, std::memory_order_relaxed);
    if (uint32_t(n) < most) cfg.gridDim = dim3(uint32_t(n) * kCluster);
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, maps, p, tokens);
    if (e != cudaSuccess) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention_mass: %s", cudaGetErrorString(e));
    return launch_status("jfb_paged_attention_mass");
}

}  // namespace

jfb_status launch_mass_tc(const jfb_paged_cache & cache, const CUtensorMap & k, MassParams p, const Device & device, cudaStream_t s) {
    const uint32_t tokens = 128 / p.view.group;
    p.view.item_rows = tokens * p.view.group;
    MassMaps maps;
    maps.k = k;
    if (!query_map(maps.q, p.view, p.q, p.q_stride, p.heads, tokens)) {
        return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention_mass: could not encode a TMA tensor map");
    }
    const bool half = cache.dtype == JFB_DTYPE_F16;
    if (cache.head_dim <= 64) return half ? launch<__half, 64>(maps, p, tokens, device, s) : launch<__nv_bfloat16, 64>(maps, p, tokens, device, s);
    return half ? launch<__half, 128>(maps, p, tokens, device, s) : launch<__nv_bfloat16, 128>(maps, p, tokens, device, s);
}

}  // namespace paged
}  // namespace jfb
