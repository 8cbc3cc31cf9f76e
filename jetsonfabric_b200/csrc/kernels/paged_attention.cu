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
// per SM). Each of the 8 consumer warps forms the scores of 16 keys of a tile;
// the probabilities meet in shared memory, and each warp forms all keys' sums
// of its D / 8 output columns. The warps share one running maximum, so the end
// of an item costs one exchange of the softmax sums. (Warps that kept their own
// maximum and sums over their own keys had 64 KB to add up at every end: 2
// more us each, of which a batch of short sequences has several per CTA.) The
// scores of the next tile are formed beside the second product of this one.
// A part of an item that began in another CTA is published by a warp of its
// own, so that the consumers go on to their next item at once.
//
// 6 sequences of 9001 to 65001 keys, 28/4 heads: 82 us (84 % of the measured
// copy bandwidth); 64 of 1025 to 1280: 37 us (63 %), of which the way to the
// first tile and the ends are a third.

constexpr int kRowsM = 16;
constexpr int kItemRows = 0;  // units of an item's start and end
constexpr int kConsumers = 8;
constexpr int kThreadsRows = (kConsumers + 3) * 32;  // and K's and V's producers, the publisher

template <int D>
struct RowsSmem {
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr uint32_t kStage = 2 * kTileBytes<D>;
    static constexpr uint32_t kP = kStages * kStage;                            // [2][16 rows][128 keys] probabilities
    static constexpr uint32_t kTops = kP + 2 * kRowsM * kTileKeys * 2;          // [8 warps][16]
    static constexpr uint32_t kSums = kTops + kConsumers * kRowsM * 4;          // [8 warps][16]
    static constexpr uint32_t kBars = kSums + kConsumers * kRowsM * 4;          // full K, full V, empty
    static constexpr uint32_t kWalk = kBars + 3 * kStages * 8;
    static constexpr uint32_t kFlags = kWalk + kThreadsRows / 32 * sizeof(Walk);  // abort, joined at once
    static constexpr uint32_t kBytes = kFlags + 16 + 1024;                        // + alignment
};
static_assert(RowsSmem<128>::kBytes <= 232448 && RowsSmem<64>::kBytes <= 232448);
static_assert(RowsSmem<64>::kP >= JFB_PAGED_MAX_SEQUENCES * 8);

__device__ __forceinline__ void bar_consumers() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// The same, and whether any of the threads brings true.
__device__ __forceinline__ bool bar_consumers_or(bool mine) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any)
                 : "r"(uint32_t(mine))
                 : "memory");
    return any != 0;
}

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

// Consumers hand the part of an item that began elsewhere to the publisher,
// and learn at the CTA's end whether it was the item's last.
__device__ __forceinline__ void part_arrive() { asm volatile("bar.arrive 2, 288;" ::: "memory"); }
__device__ __forceinline__ void part_wait() { asm volatile("bar.sync 2, 288;" ::: "memory"); }
__device__ __forceinline__ void verdict_arrive() { asm volatile("bar.arrive 3, 288;" ::: "memory"); }
__device__ __forceinline__ void verdict_wait() { asm volatile("bar.sync 3, 288;" ::: "memory"); }

// Counts a part in; true when all the item's parts are.
__device__ __forceinline__ bool count_part(uint32_t * counter, uint32_t others) {
    __threadfence();
    const bool last = atomicAdd(counter, 1u) == others;
    __threadfence();
    if (last) *counter = 0;
    return last;
}

// Where CTA c keeps its part of the item that begins in CTA c0: [16][D] sums, then [16] (maximum, sum).
__device__ __forceinline__ float * part_of(const AttentionParams & p, uint32_t c, uint32_t c0) {
    return p.partial + uint64_t(2 * c + (c == c0 ? 1 : 0)) * kSlotFloats;
}

// Adds a part (maximum, sum and N columns) to another. The operations are
// spelled out, so that every place that joins gets the same bits.
template <int N>
__device__ __forceinline__ void join_part(float & m, float & l, float (&o)[N], float pm, float pl, const float (&po)[N]) {
    const float top = fmaxf(m, pm);
    const float f = m == -INFINITY ? 0.0f : exp2_approx(m - top), g = pm == -INFINITY ? 0.0f : exp2_approx(pm - top);
    m = top;
    l = fmaf(pl, g, __fmul_rn(l, f));
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = fmaf(po[i], g, __fmul_rn(o[i], f));
}

// The consumers join all parts of the walk's item: 16 threads per row and
// slice of the parts, the slices merged in order. Where rows are few their
// parts are many (a long context of one sequence), and more slices keep more
// loads in flight. Two parts are joined in plain CTA order whatever the slices.
template <typename T, int D>
__device__ __forceinline__ void join_item(const AttentionParams & p, const Walk & w, float * scratch) {
    constexpr int kN = D / 16;  // columns per thread
    uint32_t c0, c1;
    walk_owners<kItemRows>(w, c0, c1);
    const uint32_t row0 = w.tile * kRowsM, rows = min(uint32_t(kRowsM), w.s.count * p.view.group - row0);
    const uint32_t slices = kRowsM / rows, unit = threadIdx.x >> 4, slice = unit / rows, row = unit - slice * rows;
    const uint32_t col = (threadIdx.x & 15) * kN;
    float m = -INFINITY, l = 0.0f, o[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) o[i] = 0.0f;
    if (slice < slices) {
#pragma unroll 8
        for (uint32_t c = c0 + slice; c <= c1; c += slices) {
            const float * from = part_of(p, c, c0);
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(from + kRowsM * D + 2 * row));
            float x[kN];
#pragma unroll
            for (int i = 0; i < kN; i += 4) {
                const float4 y = __ldcg(reinterpret_cast<const float4 *>(from + row * D + col + i));
                x[i] = y.x, x[i + 1] = y.y, x[i + 2] = y.z, x[i + 3] = y.w;
            }
            join_part(m, l, o, ml.x, ml.y, x);
        }
    }
    float * mine = scratch + threadIdx.x * (kN + 2);
    if (slice > 0) {
        mine[0] = m;
        mine[1] = l;
#pragma unroll
        for (int i = 0; i < kN; ++i) mine[2 + i] = o[i];
    }
    bar_consumers();
    if (slice == 0) {
        for (uint32_t s = 1; s < slices; ++s) {
            const float * other = mine + s * rows * 16 * (kN + 2);
            float x[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i) x[i] = other[2 + i];
            join_part(m, l, o, other[0], other[1], x);
        }
        const uint32_t r = row0 + row;
        const RowsOut<T> out(p, true, w.s.q0 + r / p.view.group, w.kv_head * p.view.group + r % p.view.group);
#pragma unroll
        for (int i = 0; i < kN; i += 2) out.store2(col + i, o[i], o[i + 1], l, p.view.head_dim);
        if (col == 0) out.store_lse(p, m, l);
    }
    bar_consumers();  // scratch may be written again
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

    uint32_t s0, s1;
    walk_segment<kItemRows>(w, s0, s1);
    // the CTA's first segment is a part of an item that began elsewhere, and others follow it
    const bool handed = s0 > 0 && w.item0 + w.k.tiles + 2 * kItemRows < w.end;
    if (warp == kConsumers + 2) {
        if (!handed) return;
        uint32_t c0, c1;
        walk_owners<kItemRows>(w, c0, c1);
        part_wait();
        if (lane == 0) flags[2] = count_part(p.counters + c0, c1 - c0);
        __syncwarp();
        verdict_arrive();
        return;
    }
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
            if (!is_v) {
                // the item's queries on their way to L1 before the consumers get to it: half a row per lane
                const uint32_t r = w.tile * kRowsM + lane / 2;
                if (r < w.s.count * v.group && (lane & 1) * 64 < v.head_dim) {
                    const T * src = static_cast<const T *>(p.q) + uint64_t(w.s.q0 + r / v.group) * p.q_stride +
                                    uint64_t(head * v.group + r % v.group) * v.head_dim + (lane & 1) * 64;
                    uint32_t unused;
                    asm volatile("ld.global.b32 %0, [%1];" : "=r"(unused) : "l"(src));
                }
            }
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
                tile_issue<D>(v, load, map, head, smem_u32(smem) + st * L::kStage + (is_v ? kTileBytes<D> : 0u), full + st);
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
    constexpr int kCols = D / 8;      // output columns of a warp
    constexpr int kTilesN = kCols / 8;
    const uint32_t grp = lane >> 2, tig = lane & 3;
    const uint32_t G = v.group, hd = v.head_dim;
    const float scale2 = p.scale * kLog2e;
    float * tops = reinterpret_cast<float *>(smem + L::kTops);
    float * sums = reinterpret_cast<float *>(smem + L::kSums);
    const uint32_t p_base = smem_u32(smem) + L::kP;
    uint32_t n = 0;
    do {
        uint32_t t0, t1;
        walk_segment<kItemRows>(w, t0, t1);
        const uint32_t packed = w.s.count * G;  // rows of an item: below 2^31 (checked on the host)
        const uint32_t row0 = w.tile * kRowsM;
        const int32_t first = int32_t(w.s.kv) - int32_t(w.s.count);
        // Q fragments of rows grp and grp + 8
        uint32_t qa[D / 16][4];
        int32_t pos[2];
        uint32_t out_row[2], out_head[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t r = row0 + grp + 8 * e;
            const bool valid = r < packed;
            const uint32_t i = valid ? r / G : 0u, g = valid ? r % G : 0u;
            out_row[e] = w.s.q0 + i;
            out_head[e] = w.kv_head * G + g;
            pos[e] = first + int32_t(i);
            const T * src = static_cast<const T *>(p.q) + uint64_t(out_row[e]) * p.q_stride + uint64_t(out_head[e]) * hd;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t d = kk * 16 + h * 8;
                    qa[kk][e + 2 * h] = valid && d < hd ? *reinterpret_cast<const uint32_t *>(src + d + tig * 2) : 0u;
                }
            }
        }
        const int32_t pos_first = first + int32_t(row0 / G);
        const int32_t pos_last = first + int32_t((min(row0 + uint32_t(kRowsM), packed) - 1) / G);
        float o[kTilesN][4];
#pragma unroll
        for (int j = 0; j < kTilesN; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        const int32_t begin = int32_t(w.k.begin + warp * 16), lo = int32_t(w.k.lo), hi = int32_t(w.k.hi);
        // scores of this warp's 16 keys of tile t, the a-th of the CTA; after a wait that gave up
        // no work is done, but every warp still meets the others at the barriers
        float s[2][4];
        bool live;
        const auto scores = [&](uint32_t a, uint32_t t) {
            live = !__any_sync(0xffffffffu, flags[0]) &&
                   __all_sync(0xffffffffu, mbar_wait(full_k + a % L::kStages, (a / L::kStages) & 1, flags, v.error));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
            }
            if (!live) return;
            const uint32_t kbase = smem_u32(smem) + (a % L::kStages) * L::kStage;
            const uint32_t krow = warp * 16 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                uint32_t b[4];
                const uint32_t chunk = kk * 2 + ((lane >> 3) & 1);
                ldsm4(b, kbase + (chunk >> 3) * (kTileKeys * 128) + krow * 128 + (((chunk & 7) ^ (krow & 7)) << 4));
                mma_16816<T>(s[0], qa[kk], b[0], b[1]);
                mma_16816<T>(s[1], qa[kk], b[2], b[3]);
            }
            const int32_t key = begin + int32_t(t * kTileKeys);
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
        };
        scores(n, t0);
        for (uint32_t t = t0; t < t1; ++t, ++n) {
            const uint32_t st = n % L::kStages, parity = (n / L::kStages) & 1;
            const uint32_t vbase = smem_u32(smem) + st * L::kStage + kTileBytes<D>;
            const uint32_t pbase = p_base + (n & 1) * (kRowsM * kTileKeys * 2);
            float mx[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[e] = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
                mx[e] = scaled_top(fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2)), scale2);
            }
            // The sums refer to a number that all warps share; it moves only
            // when some row's maximum has outgrown it.
            if (bar_consumers_or(outgrown<T>(mx[0], m[0]) || outgrown<T>(mx[1], m[1]))) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (tig == 0) tops[warp * kRowsM + grp + 8 * e] = mx[e];
                }
                bar_consumers();
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = -INFINITY;
#pragma unroll
                    for (int x = 0; x < kConsumers; ++x) top = fmaxf(top, tops[x * kRowsM + grp + 8 * e]);
                    if (outgrown<T>(top, m[e])) {
                        const float next = top - kHeadroom<T>, f = exp2_approx(m[e] - next);
                        m[e] = next;
                        l[e] *= f;
#pragma unroll
                        for (int j = 0; j < kTilesN; ++j) {
                            o[j][2 * e] *= f;
                            o[j][2 * e + 1] *= f;
                        }
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float base = m[e] == -INFINITY ? 0.0f : m[e];  // nothing seen yet: every term is 0
                float q[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) q[c] = exp2_approx(fmaf(s[c >> 1][2 * e + (c & 1)], scale2, -base));
                l[e] += (q[0] + q[1]) + (q[2] + q[3]);
                // 16-byte chunks 2 warp and 2 warp + 1 of the row's 128 keys, chunk c at c ^ (row % 8)
                const uint32_t row = grp + 8 * e, at = pbase + row * (kTileKeys * 2) + tig * 4;
                const uint32_t c0 = (2 * warp) ^ (row & 7), c1 = (2 * warp + 1) ^ (row & 7);
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + c0 * 16), "r"(Num<T>::pack(q[0], q[1])) : "memory");
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + c1 * 16), "r"(Num<T>::pack(q[2], q[3])) : "memory");
            }
            const bool ready = live && __all_sync(0xffffffffu, mbar_wait(full_v + st, parity, flags, v.error));
            // what no row sees may hold anything: its probability is 0, but 0 x NaN is not
            const int32_t key = begin + int32_t(t * kTileKeys);
            if (ready && (key < lo || key + 16 > hi)) {
                const int32_t from = max(0, min(16, lo - key)), to = max(0, min(16, hi - key));  // rows [from, to) stay
                for (int32_t i = int32_t(lane); i < 16 * (D / 8); i += 32) {
                    const int32_t r = i / (D / 8), c = i % (D / 8);
                    if (r < from || r >= to) {
                        const uint32_t at = vbase + (c >> 3) * (kTileKeys * 128) + (warp * 16 + r) * 128 + ((c & 7) << 4);
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
                    }
                }
                fence_proxy_async();  // before the copy that reuses the stage
            }
            bar_consumers();
            if (t + 1 < t1) scores(n + 1, t + 1);
            if (!ready) continue;
#pragma unroll
            for (int kk = 0; kk < kTileKeys / 16; ++kk) {
                uint32_t a[4], b[4];
                const uint32_t arow = lane & 15;
                ldsm4(a, pbase + arow * (kTileKeys * 2) + (((2 * kk + (lane >> 4)) ^ (arow & 7)) << 4));
                const uint32_t vrow = kk * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
                const uint32_t chunk = warp * kTilesN + (kTilesN == 2 ? lane >> 4 : 0u);
                ldsm4_trans(b, vbase + (chunk >> 3) * (kTileKeys * 128) + vrow * 128 + (((chunk & 7) ^ (vrow & 7)) << 4));
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) mma_16816<T>(o[j], a, b[2 * j], b[2 * j + 1]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + st);
        }

        // the softmax sums of all keys
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
            if (tig == 0) sums[warp * kRowsM + grp + 8 * e] = l[e];
        }
        bar_consumers();
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[e] = 0.0f;
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) l[e] += sums[x * kRowsM + grp + 8 * e];
        }
        bool write = t0 == 0 && t1 == w.k.tiles;
        bool join = false;
        if (!write) {
            // One part of an item that spans CTAs: the last CTA to get here joins
            // all. With two parts that is mostly the CTA that began the item, at
            // its end: it finds the other's there and keeps its own in registers.
            uint32_t c0, c1;
            walk_owners<kItemRows>(w, c0, c1);
            if (t0 == 0 && c1 == c0 + 1) {
                if (threadIdx.x == 0) {
                    uint32_t there;
                    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(there) : "l"(p.counters + c0) : "memory");
                    flags[1] = there;
                    if (there) p.counters[c0] = 0;  // nobody else is left to arrive
                }
                bar_consumers();
                write = flags[1] != 0;
            }
            if (write) {
                const float * from = part_of(p, c1, c0);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t row = grp + 8 * e;
                    const float2 ml = __ldcg(reinterpret_cast<const float2 *>(from + kRowsM * D + 2 * row));
                    float mine[2 * kTilesN], x[2 * kTilesN];
#pragma unroll
                    for (int j = 0; j < kTilesN; ++j) {
                        const float2 y = __ldcg(reinterpret_cast<const float2 *>(from + row * D + warp * kCols + j * 8 + tig * 2));
                        x[2 * j] = y.x;
                        x[2 * j + 1] = y.y;
                        mine[2 * j] = o[j][2 * e];
                        mine[2 * j + 1] = o[j][2 * e + 1];
                    }
                    join_part(m[e], l[e], mine, ml.x, ml.y, x);
#pragma unroll
                    for (int j = 0; j < kTilesN; ++j) {
                        o[j][2 * e] = mine[2 * j];
                        o[j][2 * e + 1] = mine[2 * j + 1];
                    }
                }
            } else {
                float * to = part_of(p, blockIdx.x, c0);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t row = grp + 8 * e;
#pragma unroll
                    for (int j = 0; j < kTilesN; ++j) {
                        __stcg(reinterpret_cast<float2 *>(to + row * D + warp * kCols + j * 8 + tig * 2), make_float2(o[j][2 * e], o[j][2 * e + 1]));
                    }
                    if (warp == 0 && tig == 0) __stcg(reinterpret_cast<float2 *>(to + kRowsM * D + 2 * row), make_float2(m[e], l[e]));
                }
                if (handed && t0 > 0) {
                    part_arrive();
                } else {  // the CTA's last segment
                    bar_consumers();
                    if (threadIdx.x == 0) flags[1] = count_part(p.counters + c0, c1 - c0);
                    bar_consumers();
                    join = flags[1] != 0;
                }
            }
        }
        if (join) join_item<T, D>(p, w, reinterpret_cast<float *>(smem));  // the ring is idle: no segment follows
        if (write) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const RowsOut<T> out(p, row0 + grp + 8 * e < packed, out_row[e], out_head[e]);
#pragma unroll
                for (int j = 0; j < kTilesN; ++j) out.store2(warp * kCols + j * 8 + tig * 2, o[j][2 * e], o[j][2 * e + 1], l[e], hd);
                if (warp == 0 && tig == 0) out.store_lse(p, m[e], l[e]);
            }
        }
    } while (walk_warp_next<kItemRows>(v, &w));
    if (handed) {
        verdict_wait();
        if (flags[2]) join_item<T, D>(p, walks[kConsumers + 2], reinterpret_cast<float *>(smem));
    }
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

// The tcgen05 kernel takes 128 packed rows at once and 10 us more for its start
// and end, the other 16: from 2 row tiles of 16 a sequence on, if there is work
// for it, counted in (16 rows, 128 keys) tiles of the keys that the table can
// hold. Rows kernel / tcgen05 kernel at 28/4 heads, in us: 64 sequences of
// 1025 to 1280 keys with 2, 4, 6, 8 new tokens 39/50, 64/50, 88/51, 113/52;
// one of 1000 keys with 8, 16, 48 tokens 13/20, 13/20, 19/24 (672 tiles); 4 of them with
// 16, 24, 40, 48: 20/20, 24/22, 33/24 (2240), 40/24 (2688); one of 8000 with 8, 16, 48: 21/32,
// 28/32, 54/41 (5292). The few-rows kernel is kept where that is not much.
//
// The host knows neither the lengths nor how the rows divide among the
// sequences (a captured call serves others). So the keys are the table's width,
// which costs a short context in a wide table up to the difference above (one
// of 1000 keys with 8 tokens: 13 us, 20 in a table 128 times as wide), and one
// kernel serves all sequences by their mean: 63 single tokens (37 us by
// themselves) with a chunk of 220 over 8000 keys (50) take 258 us on the
// few-rows kernel, with one of 512 (70) 108 on the other.
extern "C" int jfb_paged_attention_uses_tiles(uint32_t rows, uint32_t heads, uint32_t window, const jfb_paged_cache * cache,
                                              const jfb_paged_batch * batch) {
    const uint32_t group = heads / cache->kv_heads;
    uint64_t keys = uint64_t(batch->table_width) * cache->page_size;
    if (window > 0) keys = std::min(keys, uint64_t(window) + rows / batch->sequences);
    const double tiles = double((uint64_t(rows) * group + 15) / 16) * cache->kv_heads * double((keys + kTileKeys - 1) / kTileKeys);
    return group <= 128 && uint64_t(rows) * group > 32ull * batch->sequences && tiles > 2500;
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
    if (!(scale > 0.0f) || scale > 1.0e38f || window > 0x7fffffffu) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_attention needs a positive scale up to 1e38 and a window below 2^31");
    }
    if (rows == 0 || batch->sequences == 0) return status_ok();
    // one item's results would replace queries that another has still to read
    if (rows_overlap(q, q_stride, out, out_stride, rows, uint64_t(heads) * cache->head_dim)) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "jfb_paged_attention: q and out overlap");
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
    if (jfb_paged_attention_uses_tiles(rows, heads, window, cache, batch)) return launch_attention_tc(*cache, mk, mv, p, device, s);
    if (cache->head_dim <= 64) {
        return half ? launch_rows<__half, 64>(mk, mv, p, device, s) : launch_rows<__nv_bfloat16, 64>(mk, mv, p, device, s);
    }
    return half ? launch_rows<__half, 128>(mk, mv, p, device, s) : launch_rows<__nv_bfloat16, 128>(mk, mv, p, device, s);
}
