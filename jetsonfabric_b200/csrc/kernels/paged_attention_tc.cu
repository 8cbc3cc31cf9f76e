// Attention of chunks over a cache in pages on the tcgen05 tensor cores.
//
// An item is two row tiles of one sequence and kv head, each the packed rows
// (token, head of the group) of 128 / G whole tokens, so that the tile's
// queries are one box of TMA; its keys come in tiles of 128. One CTA per SM
// walks its share of the units (walk_begin):
//   warps 0-3, 4-7  softmax of row tile 0 and 1, a thread per row: scores from
//                   tensor memory, running maximum and sum, probabilities back
//                   as the 16-bit A operand, results out;
//   warps 8, 11     the MMAs, S_x = Q_x K^T from one and O_x += P_x V from the
//                   other, each waiting only for what its own chain needs;
//   warps 9, 10     K and V tiles, page by page through TMA (one warp for both
//                   was slower where pages are small, a copy per page and 64
//                   columns: 104 us against 93 for chunks of 65 to 519 tokens at
//                   16 tokens a page, 90 against 90 at 64); 10 also the queries of
//                   the next item, as soon as the last scores of this one are formed.
// K and V have a ring each. In one ring of five tiles a slot would hold them by
// turns, and the warp that waits for K alone, by parity, could take the end of
// an earlier phase than the V tile's, still on its way, for its own.
// Tensor memory (512 columns): O_0 and O_1 of 128 f32 columns, P_0 and P_1 of
// 64 columns of 16-bit pairs, and one S of 128. The row tiles take turns with
// S: a softmax thread moves its row into registers at once, which frees S for
// the other tile's scores while it works, so the scores a row tile needs next
// are formed during its current exponentials.
//
// O is rescaled only when a row's maximum has grown by more than 2^8 over the
// one its sums refer to (the sums stay far inside f32's range, the probabilities
// inside their type's), so most tiles touch O not at all.
//
// Two row tiles of a key tile need the tensor pipe (four products of 128 x 128
// x 128 at 8192 operations a cycle) and the exponentials' unit (16 a cycle) for
// 2048 cycles each: neither alone bounds the time, but a row tile's products and
// exponentials follow one another, and with one S between the two row tiles they
// overlap only in part. A prompt of 8192 at 28/4 heads, 397,000 cycles of both
// (209 us at 1.9 GHz), takes 426 us after a pause and 471 to 478 (1010 TFLOP/s
// of the measured 1665) in long runs, where the power cap leaves 1.62 GHz.
#include "paged_attention.cuh"
#include "paged_tc.cuh"

namespace jfb {
namespace paged {
namespace {

// Units of an item's start and end (a prompt of 8192, 28/4 heads: 449, 409, 388,
// 389 us with 1 to 4, before K and V had a ring each).
constexpr int kItemTc = 3;
// A part's joining in sixteenths of a unit, which bounds the parts of an item.
// One chunk of 16 tokens over 8000 keys, 28/4 heads: 60 us when every SM took
// a part, and 45, 37, 34, 33 us with 64, 32, 16, 8; 41 with 2 (over 30000 keys
// 67, and 75, 62, 56, 54, 62). Unrolling the join's loop over the parts did not
// help: its code runs once, and costs more to fetch than the loads' latency.
constexpr uint32_t kJoinTc = 8;
// What the parts at a CTA's start and end cost it, in units: up to that much
// imbalance, items are not cut.
constexpr uint32_t kPartsTc = 12;
constexpr int kThreadsTc = 384;
constexpr int kWarpS = 8, kWarpK = 9, kWarpV = 10;  // warp 11 issues P V
constexpr uint32_t kColO = 0, kColP = 256, kColS = 384;  // O_1 is 128 and P_1 64 columns further

template <int D>
struct TcSmem {
    // the rings, one after the other (3 and 2: a prompt of 8192 at 28/4 heads 416 us, 411 with 2 and 3)
    static constexpr int kStagesK = D == 128 ? 2 : 5, kStagesV = D == 128 ? 3 : 5;
    static constexpr int kStages = kStagesK + kStagesV;
    static constexpr uint32_t kQ = 2 * kTileBytes<D>;
    static constexpr uint32_t kBars = kQ + kStages * kTileBytes<D>;
    static constexpr uint32_t kNumBars = 2 * kStages + 11;  // full, empty; s, p, o, q full and q free of both row tiles; S free
    static constexpr uint32_t kWalk = kBars + kNumBars * 8;
    static constexpr uint32_t kFlags = kWalk + kThreadsTc / 32 * sizeof(Walk);  // abort, last of tile 0 and 1, tmem
    static constexpr uint32_t kBytes = kFlags + 32;
};
static_assert(TcSmem<128>::kBytes <= 232448 && TcSmem<64>::kBytes <= 232448);
static_assert(TcSmem<64>::kBars >= JFB_PAGED_MAX_SEQUENCES * 8);

// First token of row tile x of the walk's item, and whether the item has a second one.
__device__ __forceinline__ uint32_t first_token(const Walk & w, uint32_t tokens, uint32_t x) { return (w.tile * 2 + x) * tokens; }
__device__ __forceinline__ bool two_tiles(const Walk & w, uint32_t tokens) { return w.s.count > first_token(w, tokens, 1); }

// The calling warp zeroes rows [a, b) of a tile (a <= b <= 128).
template <int D>
__device__ __forceinline__ void clear_rows(uint32_t tile, uint32_t a, uint32_t b) {
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t i = a * 8 + lane; i < b * 8; i += 32) {
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + h * kHalfBytes + i * 16), "r"(0) : "memory");
        }
    }
}

// The 128 threads of one row tile's softmax.
__device__ __forceinline__ void bar_tile(uint32_t x) {
    if (x == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
    else asm volatile("bar.sync 2, 128;" ::: "memory");
}

struct TcMaps {
    CUtensorMap k, v, q;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreadsTc, 1) paged_tc_kernel(const __grid_constant__ TcMaps maps, const AttentionParams p,
                                                                 const uint32_t tokens, const bool sectors) {
    extern __shared__ __align__(1024) uint8_t smem[];
    using L = TcSmem<D>;
    uint64_t * full = reinterpret_cast<uint64_t *>(smem + L::kBars);
    uint64_t * empty = full + L::kStages;
    uint64_t * s_full = empty + L::kStages;
    uint64_t * p_full = s_full + 2;
    uint64_t * o_full = p_full + 2;
    uint64_t * q_full = o_full + 2;
    uint64_t * q_free = q_full + 2;
    uint64_t * s_free = q_free + 2;
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
            mbar_init(q_full + x, 1);
            mbar_init(q_free + x, 1);
        }
        mbar_init(s_free, 4);
        flags[0] = 0;
        mbar_init_fence();
    }
    pdl_trigger();
    pdl_wait();
    const View & v = p.view;
    if ((smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need it
        if (threadIdx.x == 0) flag_error(v.error, JFB_PAGED_ERROR_TIMEOUT);
        return;
    }
    Walk * walks = reinterpret_cast<Walk *>(smem + L::kWalk);
    if (!walk_begin<kItemTc, kJoinTc, kPartsTc>(v, reinterpret_cast<uint64_t *>(smem), walks)) return;
    Walk & w = walks[warp];
    __syncthreads();
    // rows that no query fills stay zero (and this may have held the walk's scratch)
    for (uint32_t i = threadIdx.x; i < L::kQ / 16; i += kThreadsTc) reinterpret_cast<uint4 *>(smem)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async();
    if (warp == kWarpS) tmem_alloc(tmem_slot);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t ring = smem_u32(smem) + L::kQ;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        bool ok = true;
        auto wait = [&](uint64_t * bar, uint32_t parity) {
            ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, flags, v.error));
            return ok;
        };
        if (warp == kWarpK || warp == kWarpV) {
            const uint32_t is_v = warp == kWarpV ? 1 : 0;
            const CUtensorMap * map = is_v ? &maps.v : &maps.k;
            const uint32_t stages = is_v ? L::kStagesV : L::kStagesK, slot0 = is_v ? L::kStagesK : 0;
            uint32_t n = 0, items[2] = {0, 0};
            do {
                uint32_t t0, t1;
                walk_segment<kItemTc>(w, t0, t1);
                const int32_t * row = v.table + uint64_t(w.b) * v.table_stride;
                const uint32_t begin = w.k.begin, kv = w.s.kv, head = w.kv_head;
                auto pages_of = [&](uint32_t t) {
                    const uint32_t key0 = begin + t * kTileKeys;
                    return tile_pages(v, row, key0, kv <= key0 ? key0 : min(kv, key0 + uint32_t(kTileKeys)));
                };
                TileLoad next = pages_of(t0);
                const uint32_t queries = is_v ? (two_tiles(w, tokens) ? 2 : 1) : 0;
                for (uint32_t x = 0; x < queries; ++x) {
                    if (items[x] > 0 && !wait(q_free + x, (items[x] - 1) & 1)) break;
                    ++items[x];
                    if (lane == 0) {
                        mbar_arrive_expect_tx(q_full + x, tokens * v.group * D * 2);
                        for (int h = 0; h < D / 64; ++h) {
                            tma_load_rows(smem_u32(smem) + x * kTileBytes<D> + h * kHalfBytes, &maps.q, h * 64, int32_t(w.kv_head * v.group),
                                          int32_t(w.s.q0 + first_token(w, tokens, x)), q_full + x);
                        }
                    }
                    __syncwarp();
                }
                for (uint32_t t = t0; ok && t < t1; ++t, ++n) {
                    const TileLoad load = next;
                    if (t + 1 < t1) next = pages_of(t + 1);
                    const uint32_t turn = n / stages, st = slot0 + n - turn * stages;
                    if (turn > 0 && !wait(empty + st, (turn - 1) & 1)) break;
                    tile_issue<D>(v, load, map, head, ring + st * kTileBytes<D>, full + st);
                }
            } while (ok && walk_warp_next<kItemTc>(v, &w));
            if (flags[0]) {
                for (uint32_t i = n > stages ? n - stages : 0u; i < n; ++i) mbar_drain(full + slot0 + i % stages, (i / stages) & 1);
                for (uint32_t x = 0; x < 2; ++x) {
                    if (items[x] > 0) mbar_drain(q_full + x, (items[x] - 1) & 1);
                }
            }
        } else {
            // steps j of a segment are (key tile j >> two, row tile j & two)
            const bool scores = warp == kWarpS;
            const uint32_t q_addr = smem_u32(smem);
            uint32_t tiles[2] = {0, 0}, items[2] = {0, 0};
            uint32_t g = 0;      // key tiles before this segment
            uint32_t moved = 0;  // times S was used
            const uint32_t stages = scores ? L::kStagesK : L::kStagesV, slot0 = scores ? 0 : L::kStagesK;
            auto full_of = [&](uint32_t n) { return wait(full + slot0 + n % stages, (n / stages) & 1); };
            do {
                uint32_t t0, t1;
                walk_segment<kItemTc>(w, t0, t1);
                const uint32_t two = two_tiles(w, tokens) ? 1 : 0;
                const uint32_t steps = (t1 - t0) << two;
                const uint32_t begin = w.k.begin, kv = w.s.kv;
                // first slot that the sequence's first new row sees
                const uint32_t seen_from = v.window > 0 && kv > w.s.count + (v.window - 1) ? kv - w.s.count - (v.window - 1) : 0u;
                for (uint32_t j = 0; j < steps; ++j) {
                    const uint32_t x = j & two, n = g + (j >> two), st = slot0 + n % stages;
                    const uint32_t addr = ring + st * kTileBytes<D>;
                    if (scores) {
                        if (x == 0 && !full_of(n)) break;
                        if (j <= two && !wait(q_full + x, items[x]++ & 1)) break;
                        if (moved > 0 && !wait(s_free, (moved - 1) & 1)) break;
                        ++moved;
                        tc_fence_after();
                        mma_scores<T, D>(tmem + kColS, q_addr + x * kTileBytes<D>, addr);
                        mma_commit(s_full + x);
                        if (j + two >= steps - 1) mma_commit(q_free + x);
                    } else {
                        const uint32_t t = t0 + (j >> two);
                        if (x == 0) {
                            if (!full_of(n)) break;
                            // Slots that no row of the sequence sees may hold anything: their
                            // probability is 0, but 0 x NaN is not.
                            const uint32_t key0 = begin + t * kTileKeys;
                            const uint32_t from = key0 < seen_from ? min(seen_from - key0, uint32_t(kTileKeys)) : 0u;
                            const uint32_t to = kv > key0 ? min(kv - key0, uint32_t(kTileKeys)) : 0u;
                            if (from > 0 || to < uint32_t(kTileKeys)) {
                                clear_rows<D>(addr, 0, from);
                                clear_rows<D>(addr, to, kTileKeys);
                                fence_proxy_async();
                                __syncwarp();
                            }
                        }
                        if (!wait(p_full + x, tiles[x]++ & 1)) break;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 0; kk < kTileKeys / 16; ++kk) {
                            mma_ts(tmem + kColO + x * 128, tmem + kColP + x * 64 + kk * 8, desc_mn_major(addr + kk * 2048),
                                   instr_desc<T>(D, true), t > t0 || kk > 0);
                        }
                        mma_commit(o_full + x);
                    }
                    if (x == two) mma_commit(empty + st);
                }
                g += t1 - t0;
            } while (ok && walk_warp_next<kItemTc>(v, &w));
            if (flags[0]) {  // MMAs in flight finish before tensor memory is given back
                const uint64_t t = global_ns();
                while (global_ns() - t < 10000000ull) __nanosleep(1000);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const uint32_t x = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = tmem + ((warp & 3) << 21);  // this warp's 32 lanes
        const uint32_t t_s = lanes + kColS, t_p = lanes + kColP + x * 64, t_o = lanes + kColO + x * 128;
        const float scale2 = p.scale * kLog2e;
        const uint32_t token = row / v.group, head = row - token * v.group;  // within the tile and the group
        uint32_t n = 0;                                                      // tiles of this row tile so far
        bool more = true;
        do {
            if (x == 1 && !two_tiles(w, tokens)) {
                more = walk_warp_next<kItemTc>(v, &w);
                continue;
            }
            uint32_t t0, t1;
            walk_segment<kItemTc>(w, t0, t1);
            const uint32_t token0 = first_token(w, tokens, x);
            const int32_t pos_first = int32_t(int64_t(w.s.kv) - w.s.count + token0), pos = pos_first + int32_t(token);
            const int32_t pos_last = pos_first + int32_t(min(tokens, w.s.count - token0)) - 1;
            const uint32_t begin = w.k.begin;
            float m = -INFINITY, l0 = 0.0f, l1 = 0.0f;
            for (uint32_t t = t0; t < t1; ++t, ++n) {
                // after a wait that gave up the tiles are skipped; the warps still meet at the barriers below
                if (__any_sync(0xffffffffu, flags[0]) || !__all_sync(0xffffffffu, mbar_wait(s_full + x, n & 1, flags, v.error))) continue;
                tc_fence_after();
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(t_s + c * 32, s + c * 32);
                tmem_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free);
                const int32_t key0 = int32_t(begin + t * kTileKeys);
                if (key0 + kTileKeys - 1 > pos_first || (v.window > 0 && key0 <= pos_last - int32_t(v.window))) {
                    const int32_t hi = pos - key0, lo = v.window > 0 ? hi - int32_t(v.window) : -1;
#pragma unroll
                    for (int i = 0; i < 128; ++i) s[i] = i <= hi && i > lo ? s[i] : -INFINITY;
                }
                float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i + 8 <= 128; i += 8) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[i + e], s[i + 4 + e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], s[124 + e]);
                const float top = scaled_top(fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]), scale2);
                // P and O are free again when the previous product is done
                if (t > t0) {
                    if (!__all_sync(0xffffffffu, mbar_wait(o_full + x, (n - 1) & 1, flags, v.error))) continue;
                    tc_fence_after();
                }
                const bool grow = outgrown<T>(top, m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float next = grow ? top - kHeadroom<T> : m;
                    const float f = grow ? exp2_approx(m - next) : 1.0f;
                    m = next;
                    l0 *= f;
                    l1 *= f;
                    if (t > t0) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            float o[16];
                            tmem_ld16(t_o + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] *= f;
                            tmem_st16(t_o + c, reinterpret_cast<const uint32_t *>(o));
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
                    tmem_st16(t_p + c * 16, pk);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + x);
            }
            // the segment's results
            const float sum = l0 + l1;
            const bool whole = t0 == 0 && t1 == w.k.tiles;
            const RowsOut<T> out(p, token < min(tokens, w.s.count - token0), w.s.q0 + token0 + token, w.kv_head * v.group + head);
            // parts are stored as [4 columns][row] so that a warp's stores are contiguous
            float * slot = p.partial + uint64_t(2 * blockIdx.x + (t0 == 0 ? 1 : 0)) * kSlotFloats;
            if (__all_sync(0xffffffffu, flags[0] == 0 && mbar_wait(o_full + x, (n - 1) & 1, flags, v.error))) {
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < D; c += 64) {
                    float o[64];
                    tmem_ld32(t_o + c, o);
                    tmem_ld32(t_o + c + 32, o + 32);
                    tmem_wait_ld();
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 64; i += 16) out.store16(c + i, o + i, sum, v.head_dim, sectors);
                    } else {
#pragma unroll
                        for (int i = 0; i < 64; i += 4) {
                            __stcg(reinterpret_cast<float4 *>(slot) + ((c + i) / 4) * 256 + x * 128 + row,
                                   make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]));
                        }
                    }
                }
                if (whole) out.store_lse(p, m, sum);
                else __stcg(reinterpret_cast<float2 *>(slot + 256 * D) + x * 128 + row, make_float2(m, sum));
            }
            tc_fence_before();
            if (!whole) {
                // the last CTA of the item to arrive joins this row tile's parts, in CTA order
                uint32_t c0, c1;
                walk_owners<kItemTc>(w, c0, c1);
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
                    auto ml_of = [&](uint32_t c) { return __ldcg(reinterpret_cast<const float2 *>(part_of(c) + 256 * D) + x * 128 + row); };
                    float jtop = -INFINITY, jsum = 0.0f;
                    for (uint32_t c = c0; c <= c1; ++c) jtop = fmaxf(jtop, ml_of(c).x);
                    for (uint32_t c = c0; c <= c1; ++c) {
                        const float2 a = ml_of(c);
                        jsum = fmaf(a.y, a.x == -INFINITY ? 0.0f : exp2_approx(a.x - jtop), jsum);
                    }
#pragma unroll 1
                    for (int d = 0; d < D; d += 64) {
                        float acc[64];
#pragma unroll
                        for (int i = 0; i < 64; ++i) acc[i] = 0.0f;
                        for (uint32_t c = c0; c <= c1; ++c) {
                            const float a = ml_of(c).x;
                            const float f = a == -INFINITY ? 0.0f : exp2_approx(a - jtop);
                            const float4 * from = reinterpret_cast<const float4 *>(part_of(c)) + (d / 4) * 256 + x * 128 + row;
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float4 y = __ldcg(from + i * 256);
                                acc[4 * i] = fmaf(y.x, f, acc[4 * i]);
                                acc[4 * i + 1] = fmaf(y.y, f, acc[4 * i + 1]);
                                acc[4 * i + 2] = fmaf(y.z, f, acc[4 * i + 2]);
                                acc[4 * i + 3] = fmaf(y.w, f, acc[4 * i + 3]);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 64; i += 16) out.store16(d + i, acc + i, jsum, v.head_dim, sectors);
                    }
                    out.store_lse(p, jtop, jsum);
                }
                bar_tile(x);
            }
            more = walk_warp_next<kItemTc>(v, &w);
        } while (more);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kWarpS) tmem_free(tmem);
}

template <typename T, int D>
jfb_status launch(const TcMaps & maps, const AttentionParams & p, uint32_t tokens, const Device & device, cudaStream_t s) {
    // rows of whole 32-byte sectors
    const bool sectors = ((reinterpret_cast<uintptr_t>(p.out) | p.out_stride * 2 | p.view.head_dim * 2) & 31u) == 0;
    cudaError_t e = allow_smem<paged_tc_kernel<T, D>>(device, TcSmem<D>::kBytes);
    if (e == cudaSuccess) e = launch_k(paged_tc_kernel<T, D>, dim3(device.sms), dim3(kThreadsTc), TcSmem<D>::kBytes, s, maps, p, tokens, sectors);
    if (e != cudaSuccess) return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention: %s", cudaGetErrorString(e));
    return launch_status("jfb_paged_attention");
}

}  // namespace

jfb_status launch_attention_tc(const jfb_paged_cache & cache, const CUtensorMap & k, const CUtensorMap & v, AttentionParams p,
                               const Device & device, cudaStream_t s) {
    const uint32_t tokens = 128 / p.view.group;
    p.view.item_rows = 2 * tokens * p.view.group;
    TcMaps maps;
    maps.k = k;
    maps.v = v;
    if (!query_map(maps.q, p.view, p.q, p.q_stride, p.heads, tokens)) {
        return status_error(JFB_STATUS_CUDA_ERROR, "jfb_paged_attention: could not encode a TMA tensor map");
    }
    const bool half = cache.dtype == JFB_DTYPE_F16;
    if (cache.head_dim <= 64) return half ? launch<__half, 64>(maps, p, tokens, device, s) : launch<__nv_bfloat16, 64>(maps, p, tokens, device, s);
    return half ? launch<__half, 128>(maps, p, tokens, device, s) : launch<__nv_bfloat16, 128>(maps, p, tokens, device, s);
}

}  // namespace paged
}  // namespace jfb
