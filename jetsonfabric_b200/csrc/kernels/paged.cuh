// Shared parts of the paged KV-cache kernels: the view of cache and batch that
// kernels take, host checks, TMA maps over pages, bounded barrier waits, and
// the division of ragged attention work over a persistent grid.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>

#include <atomic>
#include <cstring>
#include <mutex>

#include "common.cuh"
#include "jfb/jfb_paged.h"

namespace jfb {
namespace paged {

constexpr int kTileKeys = 128;  // keys of one tile of work

// ---- kernel view ----------------------------------------------------------------

struct View {
    const int32_t * q_start;
    const int32_t * kv_len;
    const int32_t * table;
    uint64_t table_stride;
    uint64_t page_stride, token_stride, head_stride;  // elements
    uint32_t sequences, table_width;
    uint32_t pages, page_size, page_shift;
    uint32_t kv_heads, head_dim;
    uint32_t rows;       // rows of the call's row arrays
    uint32_t group;      // query heads per kv head
    uint32_t window;     // 0: none
    uint32_t item_rows;  // packed rows of one item of the attention work
    uint64_t slots;      // masses kept per sequence and kv head
    int32_t * error;
};

__device__ __forceinline__ void flag_error(int32_t * error, int32_t bit) {
    if (error != nullptr) atomicOr(error, bit);
}

// Rows [q0, q0 + count) and keys kv of one sequence, cut to the call's arrays.
struct Sequence {
    uint32_t q0, count, kv;
};

// Keys that a sequence can hold: what the table covers, and slots whose tile
// ends below 2^31 (slot arithmetic is signed).
__device__ __forceinline__ uint32_t capacity(const View & v) {
    const uint64_t cap = uint64_t(v.table_width) * v.page_size;
    return cap < 0x7ffffc00u ? uint32_t(cap) : 0x7ffffc00u;
}

__device__ __forceinline__ uint32_t cut_length(const View & v, int32_t len, bool & bad) {
    const uint32_t cap = capacity(v);
    if (len < 0) bad = true;
    const uint32_t n = len < 0 ? 0u : uint32_t(len);
    if (n > cap) bad = true;
    return n > cap ? cap : n;
}

__device__ __forceinline__ Sequence load_sequence(const View & v, uint32_t b) {
    const int32_t a = v.q_start[b], e = v.q_start[b + 1];
    bool bad = false;
    Sequence s;
    s.kv = cut_length(v, v.kv_len[b], bad);
    if (a < 0 || e < a || uint32_t(e) > v.rows) {
        bad = true;
        s.q0 = s.count = 0;
    } else {
        s.q0 = uint32_t(a);
        s.count = uint32_t(e - a);
    }
    if (bad) flag_error(v.error, JFB_PAGED_ERROR_RANGE);
    return s;
}

// ---- mbarriers and TMA -----------------------------------------------------------

constexpr uint64_t kWaitNs = 2000000000ull;  // bound of every wait
constexpr uint32_t kSuspendNs = 1000000;

__device__ __forceinline__ uint32_t smem_u32(const void * p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ void mbar_init(uint64_t * bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}

__device__ __forceinline__ void mbar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }

__device__ __forceinline__ void mbar_arrive(uint64_t * bar) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void mbar_arrive_expect_tx(uint64_t * bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(smem_u32(bar)),
                 "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ bool mbar_try_wait(uint64_t * bar, uint32_t parity, uint32_t hint_ns) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(hint_ns)
        : "memory");
    return ok != 0;
}

// False when the phase has not completed within kWaitNs (recorded in *error)
// or another thread of the CTA has given up. Waiting threads are suspended:
// spinning ones would take issue slots from the others.
__device__ __forceinline__ bool mbar_wait(uint64_t * bar, uint32_t parity, volatile int * abort_flag, int32_t * error) {
    if (mbar_try_wait(bar, parity, kSuspendNs)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
        if (mbar_try_wait(bar, parity, kSuspendNs)) return true;
        if (*abort_flag) return false;
        if (global_ns() - t0 > kWaitNs) break;
    }
    *abort_flag = 1;
    flag_error(error, JFB_PAGED_ERROR_TIMEOUT);
    return false;
}

// After an abort: waits (bounded by itself) for a copy in flight.
__device__ __forceinline__ void mbar_drain(uint64_t * bar, uint32_t parity) {
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait(bar, parity, kSuspendNs) && global_ns() - t0 < kWaitNs) {}
}

__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Box (64 elements, up to 128 tokens) of one page and head (no multicast);
// x is 0 or 64 elements: 16-byte aligned.
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap * map, int32_t x, int32_t token, int32_t head,
                                              int32_t page, uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(token), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}

// Box (64 elements, heads, rows) of query rows (no multicast); x as above.
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap * map, int32_t x, int32_t head, int32_t row,
                                              uint64_t * bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(row), "r"(smem_u32(bar))
        : "memory");
}

// Bytes of a tile of kTileKeys keys of D elements, stored as D / 64 halves of
// [key][64] in the 128-byte swizzle (16-byte chunk c of key r at c ^ (r % 8)).
template <int D>
constexpr uint32_t kTileBytes = kTileKeys * D * 2;

// A tile's load by one warp, a box (a page, or 128 keys of a larger one) per
// lane, in two steps: the page ids are asked for while the tile's place in the
// ring is still in use and looked at only when it is free.
struct TileLoad {
    int32_t page;      // of this lane's box, as the table has it
    uint32_t token;    // its first token within the page
    uint32_t boxes, step;
};

// Boxes of keys [key0, key1) (at most 128, key0 a multiple of the box) of the
// sequence whose table row is `row`.
__device__ __forceinline__ TileLoad tile_pages(const View & v, const int32_t * row, uint32_t key0, uint32_t key1) {
    const uint32_t lane = threadIdx.x & 31;
    TileLoad l;
    l.step = v.page_size < uint32_t(kTileKeys) ? v.page_size : uint32_t(kTileKeys);
    l.boxes = (key1 - key0 + l.step - 1) >> (v.page_shift < 7 ? v.page_shift : 7);
    const uint32_t key = key0 + lane * l.step;
    l.token = key & (v.page_size - 1);
    l.page = 0;
    if (lane < l.boxes) l.page = row[key >> v.page_shift];
    return l;
}

// Lane 0 announces the bytes, then every lane issues its boxes. A page id
// outside the pool becomes one that reads as zeros: the tensor map fills
// coordinates outside the pool.
template <int D>
__device__ __forceinline__ void tile_issue(const View & v, const TileLoad & l, const CUtensorMap * map, uint32_t head, uint32_t dst,
                                           uint64_t * bar) {
    const uint32_t lane = threadIdx.x & 31;
    if (lane == 0) mbar_arrive_expect_tx(bar, l.boxes * l.step * D * 2);
    __syncwarp();
    if (lane < l.boxes) {
        int32_t page = l.page;
        if (page < 0 || uint32_t(page) >= v.pages) {
            flag_error(v.error, JFB_PAGED_ERROR_RANGE);
            page = int32_t(v.pages);
        }
        const uint32_t to = dst + lane * l.step * 128;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
            tma_load_page(to + h * (kTileKeys * 128), map, h * 64, int32_t(l.token), int32_t(head), page, bar);
        }
    }
    __syncwarp();
}

// ---- division of the attention work ------------------------------------------------
//
// The (row, head of the group) pairs of one sequence and kv head are packed
// into rows i * G + g and cut into row tiles of item_rows; an item is one (kv head,
// sequence, row tile) with the key tiles that any of its rows sees (one for an
// item that sees none, which then writes zeros). It takes E units for its
// start and end and one per key tile. The units of all items, kv head
// outermost, form one line that the persistent CTAs divide evenly, so long
// contexts are split, short ones gathered and causal tiles balanced by the
// same rule from lengths that only the device knows. The parts of an item that
// spans CTAs are joined in CTA order by the last one to arrive.

struct KeyRange {
    uint32_t lo, hi;   // keys [lo, hi) are seen by some row of the tile
    uint32_t begin;    // first tile's first key: lo rounded down to a box
    uint32_t tiles;    // max(1, tiles of [begin, hi))
};

// Packed rows of a sequence: the host refuses calls with 2^31 or more. A
// division is a long chain of instructions before the first copy: a single
// item, as in decode, takes none.
__device__ __forceinline__ uint32_t row_tiles(const View & v, const Sequence & s) {
    const uint32_t packed = s.count * v.group;
    return packed <= v.item_rows ? (packed > 0 ? 1u : 0u) : (packed + v.item_rows - 1) / v.item_rows;
}

__device__ __forceinline__ KeyRange key_range(const View & v, const Sequence & s, uint32_t tile) {
    const uint32_t packed = s.count * v.group;
    const int32_t first = int32_t(s.kv) - int32_t(s.count);
    int32_t p0 = first, p1 = first + int32_t(s.count) - 1;
    if (packed > v.item_rows) {
        const uint32_t r0 = tile * v.item_rows;
        p0 = first + int32_t(r0 / v.group);
        if (r0 + v.item_rows < packed) p1 = first + int32_t((r0 + v.item_rows - 1) / v.group);
    }
    KeyRange k;
    k.hi = p1 < 0 ? 0u : uint32_t(p1 + 1);
    k.lo = v.window > 0 && p0 >= int32_t(v.window) ? uint32_t(p0) - v.window + 1 : 0u;
    const uint32_t box = v.page_size < uint32_t(kTileKeys) ? v.page_size : uint32_t(kTileKeys);
    k.begin = k.lo & ~(box - 1);
    k.tiles = k.hi > k.begin ? (k.hi - k.begin + kTileKeys - 1) / kTileKeys : 1u;
    return k;
}

// Items of a sequence and their parts: row tiles with their key tiles.
struct RowItems {
    using Part = KeyRange;
    static __device__ __forceinline__ uint32_t count(const View & v, const Sequence & s) { return row_tiles(v, s); }
    static __device__ __forceinline__ Part part(const View & v, const Sequence & s, uint32_t item) { return key_range(v, s, item); }
};

template <class Items>
struct WalkOf {
    uint64_t unit, end;    // this CTA's line segment still to do
    uint64_t item0;        // first unit of the current item
    uint64_t share;        // units of a CTA; the first `extra` have one more
    uint32_t extra;
    uint32_t kv_head, b, tile;
    uint32_t whole;        // the CTA does the items whose middle lies in its segment, none in parts
    Sequence s;
    typename Items::Part k;
};
using Walk = WalkOf<RowItems>;

__device__ __forceinline__ uint64_t divide(uint64_t a, uint64_t b) {
    // 64-bit divisions take hundreds of cycles
    return (a | b) >> 32 ? a / b : uint32_t(a) / uint32_t(b);
}

// The CTA that holds `unit`.
__device__ __forceinline__ uint32_t cta_of(uint64_t unit, uint64_t share, uint32_t extra) {
    const uint64_t larger = extra * (share + 1);
    return unit < larger ? uint32_t(divide(unit, share + 1)) : extra + uint32_t(divide(unit - larger, share));
}

// Key tiles [t0, t1) of the current item that this CTA does.
template <int E, class Items>
__device__ __forceinline__ void walk_segment(const WalkOf<Items> & w, uint32_t & t0, uint32_t & t1) {
    if (E > 0 && w.whole) {
        t0 = 0;
        t1 = w.k.tiles;
        return;
    }
    const uint64_t a = w.unit - w.item0, b = w.end - w.item0;
    t0 = a > E ? uint32_t(a - E) : 0u;
    t1 = b <= E ? 0u : b - E < w.k.tiles ? uint32_t(b - E) : w.k.tiles;
}

// Moves to the following item.
template <int E, class Items>
__device__ __forceinline__ void walk_item(const View & v, WalkOf<Items> & w) {
    w.unit = w.item0 = w.item0 + w.k.tiles + E;
    ++w.tile;
    while (w.tile >= Items::count(v, w.s)) {
        w.tile = 0;
        if (++w.b >= v.sequences) {
            w.b = 0;
            ++w.kv_head;
        }
        w.s = load_sequence(v, w.b);
    }
    w.k = Items::part(v, w.s, w.tile);
}

// Moves to the CTA's next segment with tiles; false at the end of its line.
template <int E, class Items>
__device__ __forceinline__ bool walk_next(const View & v, WalkOf<Items> & w) {
    if (E > 0 && w.whole) {
        if (w.item0 + w.k.tiles + E >= w.end) return false;
        walk_item<E>(v, w);
        return w.item0 + (w.k.tiles + E) / 2 < w.end;
    }
    // what is left of the line, if not tiles of another item, is the start of one
    if (w.item0 + w.k.tiles + 2 * E >= w.end) return false;
    walk_item<E>(v, w);
    return true;
}

// walk_next of a warp's own copy in shared memory (registers are scarce in the
// kernels): lane 0 moves it.
template <int E, class Items>
__device__ __forceinline__ bool walk_warp_next(const View & v, WalkOf<Items> * w) {
    __syncwarp();
    int more = 0;
    if ((threadIdx.x & 31) == 0) more = walk_next<E>(v, *w);
    return __shfl_sync(0xffffffffu, more, 0) != 0;
}

// The CTAs that hold the first and the last tile of the current item.
template <int E, class Items>
__device__ __forceinline__ void walk_owners(const WalkOf<Items> & w, uint32_t & c0, uint32_t & c1) {
    c0 = cta_of(w.item0 + E, w.share, w.extra);
    c1 = cta_of(w.item0 + E + w.k.tiles - 1, w.share, w.extra);
}

// Positions `walks`, one WalkOf per warp of the CTA in shared memory, at the
// unit where the line of worker `index` of `workers` begins; unit == end when
// it has no work. All threads call it; `cost` is shared scratch of one u64 per
// sequence. Up to 128 sequences every warp works it out by itself from
// registers, one load's latency long: it precedes the first copy of a call
// that may be all latency. More go through `cost` and two CTA barriers.
//
// A part of an item costs its joining CTA time as well: with JOIN > 0, the cost
// of joining one in sixteenths of a unit, only so many workers get work that a
// share has sqrt(JOIN / 16 x the mean item's units), which makes an item's
// longest part and the joining take the least time in sum. And where items of
// much the same length leave the busiest CTA at most `PARTS` units above an
// even share, none is cut. (Many sequences have many items: neither matters.)
template <int E, class Items, uint32_t JOIN = 0, uint32_t PARTS = 0>
__device__ __forceinline__ void walk_locate(const View & v, uint64_t * cost, uint32_t index, uint32_t workers, WalkOf<Items> * walks) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    constexpr uint32_t kOwn = 4;  // sequences per lane
    const bool few = v.sequences <= 32 * kOwn;
    uint32_t longest = 0;
    const auto cost_of = [&](const Sequence & s, uint32_t i) {
        const uint32_t units = Items::part(v, s, i).tiles + E;
        if (PARTS > 0) longest = max(longest, units);
        return units;
    };
    // units of a sequence per lane; the lanes share the items of one that has many
    const auto units_of = [&](const Sequence & s) {
        const uint32_t items = Items::count(v, s);
        unsigned long long units = 0;
        if (items <= 4) {
            for (uint32_t i = 0; i < items; ++i) units += cost_of(s, i);
        }
        uint32_t many = __ballot_sync(0xffffffffu, items > 4);
        while (many != 0) {
            const int src = __ffs(many) - 1;
            many &= many - 1;
            Sequence o;
            o.q0 = 0;
            o.count = __shfl_sync(0xffffffffu, s.count, src);
            o.kv = __shfl_sync(0xffffffffu, s.kv, src);
            const uint32_t n = __shfl_sync(0xffffffffu, items, src);
            unsigned long long sum = 0;
            for (uint32_t i = lane; i < n; i += 32) sum += cost_of(o, i);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (int(lane) == src) units = sum;
        }
        return units;
    };
    Sequence own[kOwn];
    unsigned long long own_units[kOwn];
    unsigned long long per_head = 0;
    if (few) {
#pragma unroll
        for (uint32_t r = 0; r < kOwn; ++r) {
            own[r] = Sequence{0, 0, 0};
            if (r * 32 + lane < v.sequences) own[r] = load_sequence(v, r * 32 + lane);
        }
#pragma unroll
        for (uint32_t r = 0; r < kOwn; ++r) {
            own_units[r] = r * 32 < v.sequences ? units_of(own[r]) : 0ull;
            per_head += own_units[r];
        }
    } else {
        for (uint32_t base = warp * 32; base < v.sequences; base += warps * 32) {
            const uint32_t b = base + lane;
            const unsigned long long units = units_of(b < v.sequences ? load_sequence(v, b) : Sequence{0, 0, 0});
            if (b < v.sequences) cost[b] = units;
        }
        __syncthreads();
        for (uint32_t b = lane; b < v.sequences; b += 32) per_head += cost[b];
    }
    // sums of 32 bits where they fit: wide ones take several times the shuffles
    const bool narrow = __all_sync(0xffffffffu, per_head < (1u << 26));
    if (narrow) {
        per_head = __reduce_add_sync(0xffffffffu, uint32_t(per_head));
    } else {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) per_head += __shfl_xor_sync(0xffffffffu, per_head, d);
    }
    WalkOf<Items> x = {};
    const uint64_t total = uint64_t(per_head) * v.kv_heads;
    if (JOIN > 0 && few) {
        uint32_t items = 0;
#pragma unroll
        for (uint32_t r = 0; r < kOwn; ++r) items += Items::count(v, own[r]);
        items = __reduce_add_sync(0xffffffffu, items);
        if (PARTS > 0 && items > 0) {
            longest = __reduce_max_sync(0xffffffffu, longest);
            const float even = float(total) / float(workers), mean = float(per_head) / float(items);
            x.whole = ceilf(even / mean) * float(longest) <= even + float(PARTS);
        }
        if (items > 0 && !x.whole) {
            const uint32_t least = uint32_t(ceilf(sqrtf(JOIN / 16.0f * float(per_head) / float(items))));
            if (total < uint64_t(least) * workers) workers = uint32_t(total) < least ? 1u : uint32_t(total) / least;
        }
    }
    x.share = divide(total, workers);
    x.extra = uint32_t(total - x.share * workers);
    x.unit = index * x.share + min(index, x.extra);
    x.end = x.unit + x.share + (index < x.extra ? 1 : 0);
    if (JOIN > 0 && index >= workers) x.unit = x.end;
    if (x.unit < x.end) {
        unsigned long long left = x.unit;
        while (left >= per_head) {
            left -= per_head;
            ++x.kv_head;
        }
        // the first entry of a list whose running sum exceeds what is left: 32 at a time
        const auto find32 = [&](unsigned long long mine, int & src) {
            unsigned long long upto = mine;
            if (narrow) {
                uint32_t sum = uint32_t(mine);
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t o = __shfl_up_sync(0xffffffffu, sum, d);
                    if (int(lane) >= d) sum += o;
                }
                upto = sum;
            } else {
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const unsigned long long o = __shfl_up_sync(0xffffffffu, upto, d);
                    if (int(lane) >= d) upto += o;
                }
            }
            const uint32_t over = __ballot_sync(0xffffffffu, upto > left);
            src = __ffs(over) - 1;
            left -= __shfl_sync(0xffffffffu, over != 0 ? upto - mine : upto, over != 0 ? src : 31);
            return over != 0;
        };
        int src = 0;
        if (few) {
            bool found = false;
#pragma unroll
            for (uint32_t r = 0; r < kOwn; ++r) {
                if (!found && r * 32 < v.sequences && find32(own_units[r], src)) {
                    found = true;
                    x.b = r * 32 + src;
                    x.s.q0 = __shfl_sync(0xffffffffu, own[r].q0, src);
                    x.s.count = __shfl_sync(0xffffffffu, own[r].count, src);
                    x.s.kv = __shfl_sync(0xffffffffu, own[r].kv, src);
                }
            }
        } else {
            for (uint32_t base = 0; base < v.sequences; base += 32) {
                if (find32(base + lane < v.sequences ? cost[base + lane] : 0ull, src)) {
                    x.b = base + src;
                    break;
                }
            }
            x.s = load_sequence(v, x.b);
        }
        const uint32_t items = Items::count(v, x.s);
        if (items > 1) {
            for (uint32_t base = 0; base < items; base += 32) {
                if (find32(base + lane < items ? Items::part(v, x.s, base + lane).tiles + E : 0ull, src)) {
                    x.tile = base + src;
                    break;
                }
            }
        }
        x.item0 = x.unit - left;
        x.k = Items::part(v, x.s, x.tile);
    }
    if (PARTS > 0 && x.whole && x.unit < x.end) {
        // an item whose middle lies before or behind the segment is another CTA's
        if (x.item0 + (x.k.tiles + E) / 2 < x.unit) {
            if (x.item0 + x.k.tiles + E >= x.end) x.end = x.unit;
            else walk_item<E>(v, x);
        }
        if (x.item0 + (x.k.tiles + E) / 2 >= x.end) x.end = x.unit;
    }
    if (lane == 0) walks[warp] = x;
    __syncwarp();
    if (!few) {  // cost may be written again, by copies too
        fence_proxy_async();
        __syncthreads();
    }
}

// The same for CTAs that share items: at the first segment that has tiles.
// False when the CTA has no work.
template <int E, uint32_t JOIN = 0, uint32_t PARTS = 0, class Items>
__device__ __forceinline__ bool walk_begin(const View & v, uint64_t * cost, WalkOf<Items> * walks) {
    walk_locate<E, Items, JOIN, PARTS>(v, cost, blockIdx.x, gridDim.x, walks);
    WalkOf<Items> * w = walks + (threadIdx.x >> 5);
    if (w->unit >= w->end) return false;
    uint32_t t0, t1;
    walk_segment<E>(*w, t0, t1);
    return t0 < t1 || walk_warp_next<E>(v, w);
}

// ---- number types -------------------------------------------------------------------

template <typename T>
struct Num;
template <>
struct Num<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<__half2 *>(&u)); }
};
template <>
struct Num<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t u) {
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// ---- host side ------------------------------------------------------------------------

inline jfb_status check_cache(const jfb_paged_cache * c) {
    if (c == nullptr || c->k == nullptr || c->v == nullptr) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "paged cache pools are required");
    }
    if (c->dtype != JFB_DTYPE_F16 && c->dtype != JFB_DTYPE_BF16) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "paged cache dtype must be F16 or BF16");
    }
    if (c->page_size < 8 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)) != 0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "page_size %u is not a power of two from 8 to 1024", c->page_size);
    }
    if (c->head_dim < 8 || c->head_dim > 128 || c->head_dim % 8 != 0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "paged head_dim %u is not a multiple of 8 up to 128", c->head_dim);
    }
    if (c->pages == 0 || c->pages > 0x7fffffffu || c->kv_heads == 0 || c->kv_heads > 65535u) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "paged cache needs pages and kv heads");
    }
    const uint64_t strides[3] = {c->page_stride, c->token_stride, c->head_stride};
    for (uint64_t s : strides) {
        if (s == 0 || s % 8 != 0 || s >= (1ull << 39)) {
            return status_error(JFB_STATUS_INVALID_ARGUMENT, "paged cache strides must be positive multiples of 8 elements");
        }
    }
    if (c->token_stride < c->head_dim || c->head_stride < c->head_dim || c->page_stride < c->head_dim) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "paged cache strides make elements share addresses");
    }
    if ((reinterpret_cast<uintptr_t>(c->k) & 15u) != 0 || (reinterpret_cast<uintptr_t>(c->v) & 15u) != 0) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "paged cache pools must be 16-byte aligned");
    }
    return status_ok();
}

inline jfb_status check_batch(const jfb_paged_batch * b, bool rows) {
    // the arrays of no sequences need not exist
    if (b == nullptr || (b->sequences > 0 && ((rows && b->q_start == nullptr) || b->kv_len == nullptr || b->page_table == nullptr))) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "paged batch arrays are required");
    }
    if (b->sequences > JFB_PAGED_MAX_SEQUENCES) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "a paged call takes at most %d sequences", JFB_PAGED_MAX_SEQUENCES);
    }
    if (b->table_width == 0 || b->table_stride < b->table_width) {
        return status_error(JFB_STATUS_INVALID_ARGUMENT, "page_table rows hold %u of a stride of %llu", b->table_width,
                            static_cast<unsigned long long>(b->table_stride));
    }
    return status_ok();
}

inline View make_view(const jfb_paged_cache & c, const jfb_paged_batch & b, uint32_t rows, uint32_t group, uint32_t window,
                      int32_t * error) {
    View v;
    v.q_start = b.q_start;
    v.kv_len = b.kv_len;
    v.table = b.page_table;
    v.table_stride = b.table_stride;
    v.page_stride = c.page_stride;
    v.token_stride = c.token_stride;
    v.head_stride = c.head_stride;
    v.sequences = b.sequences;
    v.table_width = b.table_width;
    v.pages = c.pages;
    v.page_size = c.page_size;
    v.page_shift = uint32_t(__builtin_ctz(c.page_size));
    v.kv_heads = c.kv_heads;
    v.head_dim = c.head_dim;
    v.rows = rows;
    v.group = group;
    v.window = window;
    v.item_rows = 0;
    v.slots = 0;
    v.error = error;
    return v;
}

inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void * f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess) {
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
        }
    });
    return fn;
}

// Pool as (head_dim, token, head, page): boxes of 64 elements x min(page_size,
// 128) tokens in the 128-byte swizzle; elements beyond head_dim and pages
// beyond the pool read as zeros.
inline bool pool_map(CUtensorMap & map, const void * pool, const jfb_paged_cache & c) {
    PFN_cuTensorMapEncodeTiled_v12000 encode = tensor_map_encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[4] = {c.head_dim, c.page_size, c.kv_heads, c.pages};
    const cuuint64_t strides[3] = {c.token_stride * 2, c.head_stride * 2, c.page_stride * 2};
    const cuuint32_t box[4] = {64, c.page_size < uint32_t(kTileKeys) ? c.page_size : uint32_t(kTileKeys), 1, 1};
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    std::memset(&map, 0, sizeof(map));
    return encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void *>(pool), dims, strides, box, elem,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The current device and its SMs (0 when there is none).
struct Device {
    int index;
    uint32_t sms;
};
inline Device current_device() {
    Device d = {0, 0};
    int n = 0;
    if (cudaGetDevice(&d.index) == cudaSuccess &&
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, d.index) == cudaSuccess && n > 0) {
        d.sms = uint32_t(n);
    }
    return d;
}

// Allows `Kernel` its dynamic shared memory, once per device.
template <auto Kernel>
inline cudaError_t allow_smem(const Device & d, uint32_t bytes) {
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = d.index >= 0 && d.index < 64 ? 1ull << d.index : 0ull;
    if (bit != 0 && (done.load(std::memory_order_relaxed) & bit) != 0) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

}  // namespace paged
}  // namespace jfb
