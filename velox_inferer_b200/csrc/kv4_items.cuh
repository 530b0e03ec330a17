// How the attention kernels cut a step: items (request, kv head, tile of query rows), laid end to
// end in units of one tile of tokens, an equal run of units per block. The lengths live on the
// device, so every block finds its run itself. What an item costs beside its tiles (its queries, its
// result) counts as EXTRA more units, spread evenly over it: without them a block that met many
// short items ended long after the others (chunks of several prompts beside decoding requests: 230 us
// against 180 us).
//
// Short steps are cut by the item instead (see find_run): an item whole, or in parts of one block each.
#pragma once

#include "common.cuh"
#include "kv4.cuh"

namespace vx {

constexpr float NEG_BIG = -1e30f;   // "no score yet": finite, so that differences of it are numbers

// What a request asks of a kernel.
struct Request {
    int row0, n, kv_len, row_tiles;
    long long units;   // of one kv head
};

struct RowRange {
    int lo, hi;   // tokens any of the rows sees
};

template <int ROWS>
__device__ __forceinline__ RowRange rows_range(const Kv4AttnArgs& a, int G, int n, int kv_len, int tile) {
    RowRange x;
    x.lo = a.window > 0 ? max(0, kv_len - n + tile * ROWS / G - a.window + 1) : 0;
    x.hi = a.causal ? min(kv_len, kv_len - n + (min((tile + 1) * ROWS, n * G) - 1) / G + 1) : kv_len;
    return x;
}

template <int TILE>
__device__ __forceinline__ int tiles_of(const RowRange& x) {
    // an item that sees nothing still has one tile: its rows get zeros
    return x.hi <= x.lo ? 1 : (x.hi + TILE - 1) / TILE - x.lo / TILE;
}

// Requests with more new rows than the caller's hint, or with a number of query rows per kv head
// outside (min_rows, max_rows] (another kernel's), have no rows here. `units` is left to the caller.
template <int ROWS>
__device__ __forceinline__ Request request_of(const Kv4AttnArgs& a, int G, int b) {
    Request r;
    r.row0 = min(max(a.cu[b], 0), a.tokens);
    r.n = max(0, min(max(a.cu[b + 1], 0), a.tokens) - r.row0);
    r.kv_len = (int)min((long long)max(a.kv_lens[b], 0), (long long)a.cols * a.cache.page_size);
    if (r.n > a.max_new || (long long)r.n * G <= a.min_rows || (long long)r.n * G > a.max_rows) r.n = 0;
    r.row_tiles = (r.n * G + ROWS - 1) / ROWS;
    return r;
}

// Units of one kv head of a request, by the whole warp (the same request in every lane).
// `longest`, if given, is raised to the tiles of its longest item.
template <int ROWS, int TILE, int EXTRA>
__device__ __forceinline__ long long warp_units(const Kv4AttnArgs& a, int G, int n, int kv_len, int row_tiles, int* longest = nullptr) {
    long long sum = 0;
    for (int t = threadIdx.x & 31; t < row_tiles; t += 32) {
        const int nt = tiles_of<TILE>(rows_range<ROWS>(a, G, n, kv_len, t));
        sum += EXTRA + nt;
        if (longest != nullptr) *longest = max(*longest, nt);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}
// The same for a request per lane: a lane counts a single row tile itself, the warp together counts the others'.
template <int ROWS, int TILE, int EXTRA>
__device__ __forceinline__ long long lane_units(const Kv4AttnArgs& a, int G, int b, int& row_tiles, int& longest) {
    Request r{};
    if (b < a.requests) r = request_of<ROWS>(a, G, b);
    row_tiles = r.row_tiles;
    long long units = 0;
    if (r.row_tiles == 1) {
        const int nt = tiles_of<TILE>(rows_range<ROWS>(a, G, r.n, r.kv_len, 0));
        units = EXTRA + nt;
        longest = max(longest, nt);
    }
    uint32_t many = __ballot_sync(0xffffffffu, r.row_tiles > 1);
    while (many) {
        const int src = __ffs(many) - 1;
        many &= many - 1;
        const long long u = warp_units<ROWS, TILE, EXTRA>(a, G, __shfl_sync(0xffffffffu, r.n, src), __shfl_sync(0xffffffffu, r.kv_len, src),
                                                   __shfl_sync(0xffffffffu, r.row_tiles, src), &longest);
        if ((threadIdx.x & 31) == src) units = u;
    }
    return units;
}

// This block's run of units and the request it starts in. Called by all THREADS threads of the
// block; `red` holds THREADS / 32 words of shared memory, `found` two.
struct Run {
    long long total, begin, end, request_first;
    int blocks;    // blocks that have a run
    int request;
    int parts;     // 0: equal runs of tiles; else every item counts this many units, the parts it is cut into
};
// What of it is needed seldom, in shared memory: the kernels' loops need the registers.
struct Cut {
    long long total;
    int blocks, parts;
    int longest[32];   // (per warp)
};
// total * i / n; 64-bit divisions are slow, and most totals are small
__device__ __forceinline__ long long share(long long total, int i, int n) {
    return total < 1 << 20 ? (long long)((uint32_t)total * (uint32_t)i / (uint32_t)n) : total * i / n;   // (n < 2^12)
}
// First block whose run ends after unit u.
__device__ __forceinline__ int block_of(long long u, long long total, int n) {
    return (total < 1 << 20 ? (int)(((uint32_t)(u + 1) * (uint32_t)n + (uint32_t)total - 1) / (uint32_t)total)
                            : (int)(((u + 1) * n + total - 1) / total)) - 1;
}
template <int ROWS, int TILE, int EXTRA, int THREADS, int MIN_RUN, int JOIN>
__device__ __forceinline__ Run find_run(const Kv4AttnArgs& a, int G, long long* red, Cut& cut, long long* found) {
    static_assert(MIN_RUN > EXTRA, "a run inside an item holds one tile at least");
    constexpr int WARPS = THREADS / 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, hkv = a.cache.kv_heads;
    Run run;
    const bool once = a.requests <= THREADS;
    constexpr int ITEMS = 40;   // items are counted above the units
    int row_tiles = 0, longest = 0;
    long long first = 0, mine = 0;
    for (int base = 0; base < a.requests; base += THREADS) {
        first = lane_units<ROWS, TILE, EXTRA>(a, G, base + tid, row_tiles, longest) * hkv;
        mine += first + ((long long)row_tiles * hkv << ITEMS);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) {
        red[warp] = mine;
        cut.longest[warp] = longest;
    }
    __syncthreads();
    run.total = 0;
#pragma unroll
    for (int i = 0; i < WARPS; i++) {
        run.total += red[i];
        longest = max(longest, cut.longest[i]);
    }
    const long long items = run.total >> ITEMS;
    run.total &= (1LL << ITEMS) - 1;
    // MIN_RUN units per block at least (shorter runs cost more to join than they save), but an item each.
    const int grid = (int)gridDim.x;
    run.parts = 0;
    if (run.total < 1 << 20) {   // (64-bit divisions are slow, and most totals are small)
        const int n = (int)items, total = (int)run.total, most = max(n, total / MIN_RUN), cap = min(grid, most);
        // Estimates in units of the block that ends last: equal runs, which have parts of two items mostly (as many blocks
        // for every item where they are short); items cut alike, each part a block's; whole ones, several in a block
        // where there are more than blocks. With equal runs alone a chunk of 512 tokens took 44 us (26 whole), 256 tokens
        // behind 1792 took 50 us (42 in two parts), 24 requests that verify three tokens in a window 21 us (15 whole).
        const int each = n > 0 ? grid / n : 0;
        run.blocks = total < 8 * cap ? (each > 0 ? max(n, cap / n * n) : cap) : cap;
        const int equal = n > 0 ? total / run.blocks + 2 * EXTRA + JOIN : 0;
        const int whole = (each > 0 ? 1 : (n + grid - 1) / grid) * (longest + EXTRA);
        const int s = min(each, longest / MIN_RUN);
        const int alike = s > 1 ? (longest + s - 1) / s + EXTRA + JOIN : whole;
        if (n > 0 && min(whole, alike) <= equal) {
            run.parts = whole <= alike ? 1 : s;
            run.total = n * run.parts;
            run.blocks = min(grid, n * run.parts);
        }
    } else {
        run.blocks = (int)min((long long)grid, max(items, run.total / MIN_RUN));
    }
    if (tid == 0) {
        cut.total = run.total;
        cut.blocks = run.blocks;
        cut.parts = run.parts;
    }
    run.request = 0;
    run.request_first = run.begin = run.end = 0;
    if ((int)blockIdx.x >= run.blocks) return run;
    run.begin = share(run.total, blockIdx.x, run.blocks);
    run.end = share(run.total, blockIdx.x + 1, run.blocks);
    long long before = 0;
    for (int base = 0; base < a.requests; base += THREADS) {
        const int b = base + tid;
        long long v = once ? first : lane_units<ROWS, TILE, EXTRA>(a, G, b, row_tiles, longest) * hkv;
        if (run.parts) v = (long long)row_tiles * hkv * run.parts;
        long long x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (!once) {
            __syncthreads();
            if (lane == 31) red[warp] = run.parts ? x / run.parts << ITEMS : x;
            __syncthreads();
        }
        long long pre = before, sum = 0;
#pragma unroll
        for (int i = 0; i < WARPS; i++) {
            // (the first pass's words count both)
            const long long units = run.parts ? (red[i] >> ITEMS) * run.parts : red[i] & ((1LL << ITEMS) - 1);
            pre += i < warp ? units : 0;
            sum += units;
        }
        const long long lo = pre + x - v;
        if (run.begin >= lo && run.begin < lo + v) {
            found[0] = b;
            found[1] = lo;
        }
        before += sum;
        if (before > run.begin) break;
    }
    __syncthreads();
    run.request = (int)found[0];
    run.request_first = found[1];
    return run;
}

// Walks the items of a run, those it has a tile of. Called by whole warps.
template <int ROWS, int TILE, int EXTRA>
struct Items {
    Request r;
    RowRange range;
    long long u, end, item_first;
    int b, h, rt, nt, k0, k1;
    const volatile Cut& cut;

    __device__ __forceinline__ Items(const Kv4AttnArgs& a, int G, const Run& run, const Cut& cut_)
        : u(run.begin), end(run.end), b(run.request), cut(cut_) {
        if (u >= end) return;
        load(a, G);
        const long long at = u - run.request_first;   // (64-bit divisions are slow)
        h = at < 1LL << 31 && r.units < 1LL << 31 ? (int)((uint32_t)at / (uint32_t)r.units) : (int)(at / r.units);
        item_first = run.request_first + (long long)h * r.units;
        rt = 0;
        if (const int parts = cut.parts) {
            rt = (int)(u - item_first) / parts;
            item_first += (long long)rt * parts;
        } else if (r.row_tiles > 1) {   // the row tile that holds u: 32 at a time
            const int lane = threadIdx.x & 31;
            for (;; rt += 32) {
                const int t = rt + lane;
                const int v = t < r.row_tiles ? EXTRA + tiles_of<TILE>(rows_range<ROWS>(a, G, r.n, r.kv_len, t)) : 0;
                int x = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, x, o);
                    if (lane >= o) x += y;
                }
                const uint32_t past = __ballot_sync(0xffffffffu, item_first + x > u);
                const int at = past ? __ffs(past) - 1 : 31;
                const int upto = __shfl_sync(0xffffffffu, x, at), size = __shfl_sync(0xffffffffu, v, at);
                if (past) {
                    item_first += upto - size;
                    rt += at;
                    break;
                }
                item_first += upto;
            }
        }
        enter(a, G);
        if (k0 == k1) next(a, G);
    }
    __device__ __forceinline__ void load(const Kv4AttnArgs& a, int G) {
        r = request_of<ROWS>(a, G, b);
        if (const int parts = cut.parts) {
            r.units = (long long)r.row_tiles * parts;
            return;
        }
        r.units = r.row_tiles <= 1 ? (r.row_tiles ? EXTRA + tiles_of<TILE>(rows_range<ROWS>(a, G, r.n, r.kv_len, 0)) : 0)
                                   : warp_units<ROWS, TILE, EXTRA>(a, G, r.n, r.kv_len, r.row_tiles);
    }
    __device__ __forceinline__ int size() const {
        const int parts = cut.parts;
        return parts ? parts : nt + EXTRA;
    }
    // Tiles before x of the item's units.
    __device__ __forceinline__ int tile_at(long long x, int parts) const {
        if (x <= 0) return 0;
        if (parts) {   // an item of fewer tiles has fewer parts
            const int some = min(parts, nt);
            return x >= some ? nt : (int)((uint32_t)x * (uint32_t)nt / (uint32_t)some);   // (parts < 2^12, tiles < 2^20)
        }
        if (x >= nt + EXTRA) return nt;
        // (a 64-bit division only past 2^16 tiles)
        return EXTRA == 0 ? (int)x : nt < 1 << 15 ? (int)((uint32_t)x * (uint32_t)nt / (uint32_t)(nt + EXTRA))
                                                  : (int)((unsigned long long)x * nt / (unsigned)(nt + EXTRA));
    }
    __device__ __forceinline__ void enter(const Kv4AttnArgs& a, int G) {
        range = rows_range<ROWS>(a, G, r.n, r.kv_len, rt);
        nt = tiles_of<TILE>(range);
        const int parts = cut.parts;
        k0 = tile_at(u - item_first, parts);
        k1 = tile_at(end - item_first, parts);
    }
    __device__ __forceinline__ bool more() const { return u < end; }
    __device__ __forceinline__ void next(const Kv4AttnArgs& a, int G) {
        do {
            item_first += size();
            u = item_first;
            if (u >= end) return;
            if (++rt == r.row_tiles) {
                rt = 0;
                if (++h == a.cache.kv_heads) {
                    h = 0;
                    do {   // (requests without rows have no units; there is one with units, since u < end)
                        b++;
                        load(a, G);
                    } while (r.units == 0);
                }
            }
            enter(a, G);
        } while (k0 == k1);
    }
    __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == nt; }
    // The first block whose run touches the item, and the blocks that have a tile of it (only the runs at its two ends
    // can be too short for one).
    struct Blocks {
        int first, begin, end;
    };
    __device__ __forceinline__ Blocks holders() const {
        Blocks x;
        const long long total = cut.total;
        const int blocks = cut.blocks;
        x.first = block_of(item_first, total, blocks);
        if (const int parts = cut.parts) {   // a unit is a block's (or the item is whole)
            x.begin = x.first;
            x.end = x.first + min(parts, nt) - 1;
            return x;
        }
        const int last = block_of(item_first + nt + EXTRA - 1, total, blocks);
        x.begin = x.first + (tile_at(share(total, x.first + 1, blocks) - item_first, 0) == 0 ? 1 : 0);
        x.end = last - (tile_at(share(total, last, blocks) - item_first, 0) == nt ? 1 : 0);
        return x;
    }
};

// ---- reading the cache -------------------------------------------------------------------------

__device__ __forceinline__ uint4 ldg_stream16(const uint8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ldg_stream8(const uint8_t* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ldg_stream4(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ldg_stream2(const uint8_t* p) {
    uint16_t v;
    asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}

// Eight E2M1 codes of a word -> four f16x2 (byte b holds codes 2b, 2b + 1; the first in the low half).
__device__ __forceinline__ void codes_to_f16(uint32_t word, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(word));
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Scale bytes (as seven magnitude bits) to f16, times 2^-8, exactly: the E4M3 pattern moved up seven
// places is the same number with f16's bias.
__device__ __forceinline__ uint32_t scale_pair(uint32_t word, uint32_t sel) {   // sel: the two bytes, 0x4x4y
    return (__byte_perm(word, 0, sel) << 7) & 0x3f803f80u;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// A lane's operands of one block of 16 tokens.
template <int D>
struct KRegs {
    uint32_t c[2][D / 32];   // D/4 codes of tokens g and g + 8
    uint32_t s;
};
template <int D>
struct VRegs {
    uint32_t c[2][D / 32];   // [p]: tokens 8p + 2t, 8p + 2t + 1, D/8 codes each
    uint32_t s;
};

template <int D>
__device__ __forceinline__ void load_plane(uint32_t (&c)[2][D / 32], const uint8_t* p, int lane) {
    if (D == 128) {
        const uint4 x = ldg_stream16(p + lane * 16), y = ldg_stream16(p + 512 + lane * 16);
        c[0][0] = x.x; c[0][1] = x.y; c[0][D / 32 - 2] = x.z; c[0][D / 32 - 1] = x.w;
        c[1][0] = y.x; c[1][1] = y.y; c[1][D / 32 - 2] = y.z; c[1][D / 32 - 1] = y.w;
    } else {
        const uint2 x = ldg_stream8(p + lane * 8), y = ldg_stream8(p + 256 + lane * 8);
        c[0][0] = x.x; c[0][1] = x.y;
        c[1][0] = y.x; c[1][1] = y.y;
    }
}
template <int D>
__device__ __forceinline__ void load_k(KRegs<D>& r, const uint8_t* blk, int lane) {
    if (blk == nullptr) {
#pragma unroll
        for (int i = 0; i < D / 32; i++) r.c[0][i] = r.c[1][i] = 0;
        r.s = 0;
        return;
    }
    load_plane<D>(r.c, blk, lane);
    r.s = D == 128 ? ldg_stream4(blk + 16 * D + lane * 4) : ldg_stream2(blk + 16 * D + lane * 2);
}
template <int D>
__device__ __forceinline__ void load_v(VRegs<D>& r, const uint8_t* blk, int lane) {
    if (blk == nullptr) {
#pragma unroll
        for (int i = 0; i < D / 32; i++) r.c[0][i] = r.c[1][i] = 0;
        r.s = 0;
        return;
    }
    load_plane<D>(r.c, blk + 8 * D, lane);
    // the group of lane (g, t): g where a group is one lane's 16 dimensions, g / 2 where it is two lanes'
    r.s = ldg_stream4(blk + 17 * D + (D == 128 ? lane : (lane >> 3) * 4 + (lane & 3)) * 4);
}

// log2 factor of a score: softmax scale, K's divisor, 2^8 for scale_pair's 2^-8.
__device__ __forceinline__ float score_factor(const Kv4AttnArgs& a) {
    return a.scale * 1.4426950408889634f / a.cache.k_div * 256.0f;
}
// The power of two that brings a row's largest |q| into [1, 2) (a row of zeros, or of numbers below
// 2^-100, stays as it is), as an exponent.
__device__ __forceinline__ int row_exponent(float amax) {
    return min(max((int)(__float_as_uint(amax) >> 23), 27), 227) - 127;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// acc / (sum * divisor), times scale_pair's 2^8; a row that saw nothing (sum 0) is zero.
__device__ __forceinline__ float finish(float acc, float sum, float v_div) {
    return sum > 0.0f || sum != sum ? acc / (sum * v_div) * 256.0f : 0.0f;
}

}  // namespace vx
