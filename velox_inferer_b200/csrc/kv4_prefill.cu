// Attention over the 4-bit key/value cache for many query rows (prefill chunks, wide groups), on the
// 5th-generation tensor cores.
//
// An item is 256 query rows of one (request, kv head) - new tokens times the group's query heads -
// against a run of tiles of 128 cached tokens. Per tile
//   S_w = Q_w K^T       two 128 x 128 products (kind::f16, operands in shared memory),
//   P_w = 2^(S_w - m)   in registers, one row per thread, back into tensor memory as f16,
//   O_w += P_w V        two 128 x D products (A from tensor memory),
// with w the two halves of the rows: while one half is exponentiated the other half's products run.
// K and V arrive as 4-bit codes; four warps turn each tile into f16 operands in shared memory once
// for both halves (code * scale is exact), K as rows of D (K-major), V as it lies, token rows (the
// MMA reads it MN-major, so nothing is transposed). Rows are scaled by powers of two into f16's range as
// in the decode kernel; P carries a factor 2^6 so that small probabilities stay normal, and the running
// maximum is only raised, and O rescaled, when it grows by more than 2^8 (P stays below 2^14).
//
// Roles of the 16 warps: 0-3 and 4-7 softmax of the two halves (also their Q rows and results), 8-11
// conversion, 12 issues the MMAs, 13 finds the items. Tensor memory: S_0, S_1 (P over their last 64 columns),
// O_0, O_1.
//
// What bounds it: the way of a tile through one half, scores to probabilities to product, about 3700 cycles for 2 x 1024
// cycles of MMAs (2048 rows behind 6144 tokens, 64 / 8 heads of 128: 420 us, 1140 TFLOP/s, 69 % of cuBLAS bf16).
// Without any exponentials it takes 395 us. Tried and slower: turns between the halves' exponentials, two score
// buffers of 64 columns per half (477), an issuing warp per half (486), a quarter of the exponentials as polynomials
// (448). Straight-line code in the loop is kept short: with masks in line it waited for instruction fetch (510 against 449 us).
//
// Work is cut over the blocks as in the decode kernel (kv4_items.cuh); halves of an item that several
// blocks share are parked and joined in token order by the last block to arrive.
#include "common.cuh"
#include "kv4.cuh"
#include "kv4_items.cuh"
#include "tcgen.cuh"

namespace vx {

static __device__ int g_kv4_status = 0;
enum { KV4_TIMEOUT = 7 };

constexpr int PF_ROWS = 256, PF_TILE = 128, PF_THREADS = 512;
constexpr int PF_EXTRA = 3;   // tiles' worth of an item's other costs
constexpr int PF_JOIN = 6;    // and of joining its parts

template <int D>
struct PrefillCfg {
    static constexpr int PANELS = D / 64;                 // 64 f16 = one 128-byte swizzled row
    static constexpr int KV_BYTES = PF_TILE * D * 2;      // one operand tile
    static constexpr int PANEL = PF_TILE * 128;           // bytes of a panel of 128 rows
    // V first: its descriptors have the largest strides
    static constexpr int OFF_V = 0, OFF_K = 2 * KV_BYTES, OFF_Q = 4 * KV_BYTES;
    static constexpr int OFF_BARS = OFF_Q + PF_ROWS * D * 2;
    static constexpr int SMEM = OFF_BARS + 256 + 1024;    // (aligned by hand to 1024)
    static constexpr int RING = 4;                        // items the scheduling warp is ahead
    static constexpr int PART = 128 * (D + 2);            // floats of one parked half
    static constexpr uint32_t S_COL = 0, O_COL = 256;     // of half 0; half 1: + 128 / + D
    static constexpr uint32_t P_COL = 64;                 // P inside S
};

// ---- waits that end --------------------------------------------------------------------------------
// A wait that runs out (2 s) or a block that has given up: the roles go on without waiting, every
// copy and MMA they still issue stays inside the block's own memory, and the kernel ends.
struct Waiter {
    volatile int* dead;
    __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity) const {
        if (!mbar_try_wait(bar, parity)) {
            const unsigned long long t0 = global_timer_ns();
            for (uint32_t spins = 1; !mbar_try_wait(bar, parity); spins++) {
                if ((spins & 63u) != 0) continue;
                if (*dead) break;
                if (global_timer_ns() - t0 > 2000000000ull) {
                    *dead = 1;
                    atomicExch(&g_kv4_status, KV4_TIMEOUT);
                    break;
                }
            }
        }
        __syncwarp();   // lanes leave the poll one by one; what follows may be a collective of the whole warp
    }
    // The same answer in every lane.
    __device__ __forceinline__ bool given_up() const { return __any_sync(0xffffffffu, *dead != 0); }
};

// D[128 x N] (+)= A . B, f16 operands, f32 accumulator; A from tensor memory.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Instruction descriptor of kind::f16: f32 accumulator, f16 operands, M = 128.
__device__ __forceinline__ constexpr uint32_t f16_desc(uint32_t n, bool b_mn_major) {
    return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// V as the B operand, MN-major, 128-byte swizzle: 64 dimensions per 128-byte row, token rows in groups of
// eight 1024 bytes apart, the next 64 dimensions one panel further.
__device__ __forceinline__ uint64_t smem_desc_v(uint32_t addr, uint32_t panel) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(panel >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// Two single-precision operations in one instruction.
__device__ __forceinline__ void fma2(float& x, float& y, float m, float c) {
    asm("{\n\t.reg .b64 v, m2, c2;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 m2, {%2, %2};\n\tmov.b64 c2, {%3, %3};\n\t"
        "fma.rn.f32x2 v, v, m2, c2;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "+f"(x), "+f"(y) : "f"(m), "f"(c));
}
__device__ __forceinline__ void add2(float& x, float& y, float u, float v) {
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %3};\n\t"
        "add.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(x), "+f"(y) : "f"(u), "f"(v));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Waits for this thread's tensor-memory loads; the registers of `r` pass through, so nothing that uses them can be
// moved ahead of the wait.
__device__ __forceinline__ void tc_wait_ld_of(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// An item as the roles see it.
struct PrefillItem {
    int k0, k1;              // its tiles in this block; k1 = 0: no more items
    int tile0, hi;           // first tile, end of the tokens any row sees
    int b, h, row0, first;   // request, kv head, the request's first row, first query row (token * G + head) of the item
    int rows, n, kv_len;     // query rows of the item; the request's new and all tokens
    int c_first;             // the first block whose run touches it
    int c_begin, c_end;      // the blocks that hold parts of it (equal: this one alone)
    int pad[2];
};

template <int D>
__global__ void __launch_bounds__(PF_THREADS, 1)
kv4_prefill_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using C = PrefillCfg<D>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    __shared__ long long s_red[PF_THREADS / 32], s_found[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_dead;
    __shared__ int s_last[2];
    __shared__ Cut s_cut;
    __shared__ PrefillItem s_items[C::RING];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int hkv = a.cache.kv_heads, G = a.heads / hkv, page_shift = a.cache.page_shift - 4;   // of blocks per page
    const uint32_t bars = base + C::OFF_BARS;
    auto k_full = [&](int s) { return bars + 8u * s; };
    auto k_empty = [&](int s) { return bars + 16u + 8u * s; };
    auto v_full = [&](int s) { return bars + 32u + 8u * s; };
    auto v_empty = [&](int s) { return bars + 48u + 8u * s; };
    auto q_full = [&](int w) { return bars + 64u + 8u * w; };
    auto s_full = [&](int w) { return bars + 80u + 8u * w; };
    auto p_full = [&](int w) { return bars + 96u + 8u * w; };
    auto o_full = [&](int w) { return bars + 112u + 8u * w; };
    auto o_empty = [&](int w) { return bars + 128u + 8u * w; };
    const uint32_t drained = bars + 144u;
    auto joined = [&](int w) { return bars + 232u + 8u * w; };   // the threads of a half among themselves
    auto p_half = [&](int w) { return bars + 216u + 8u * w; };   // the last 64 tokens of P
    auto item_full = [&](int i) { return bars + 152u + 8u * i; };
    auto item_empty = [&](int i) { return bars + 184u + 8u * i; };

    if (tid == 0) {
        grid_launch_dependents();
        s_dead = 0;
        for (int i = 0; i < 2; i++) {
            mbar_init(k_full(i), 4);
            mbar_init(k_empty(i), 1);
            mbar_init(v_full(i), 4);
            mbar_init(v_empty(i), 1);
            mbar_init(q_full(i), 128);
            mbar_init(s_full(i), 1);
            mbar_init(joined(i), 128);
            mbar_init(p_half(i), 128);
            mbar_init(p_full(i), 128);
            mbar_init(o_full(i), 1);
            mbar_init(o_empty(i), 128);
        }
        mbar_init(drained, 1);
        for (int i = 0; i < C::RING; i++) {
            mbar_init(item_full(i), 1);
            mbar_init(item_empty(i), 13);   // eight softmax warps, four converting, one issuing
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    grid_dependency_wait();
    const Run run = find_run<PF_ROWS, PF_TILE, PF_EXTRA, PF_THREADS, 4, PF_JOIN>(a, G, s_red, s_cut, s_found);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const Waiter wait{&s_dead};

    // every warp that works takes the items in turn; they stay in shared memory until it gives them back
    int item_no = 0;
    auto take = [&](int ahead = 0) -> const PrefillItem* {
        const int no = item_no + ahead, i = no % C::RING;
        wait(item_full(i), (uint32_t)(no / C::RING) & 1u);
        return s_items[i].k1 > 0 && !wait.given_up() ? &s_items[i] : nullptr;
    };
    auto give_back = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(item_empty(item_no % C::RING));
        item_no++;
    };

    if (warp < 8) {
        // ---------------- softmax of one half: a row per thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 160;" ::: "memory");
        const int w = warp >> 2, row = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) * 32u << 16;
        const uint32_t ts = tmem + lanes + C::S_COL + 128u * w, to = tmem + lanes + C::O_COL + (uint32_t)D * w;
        const float soft = score_factor(a);
        uint32_t* tickets = reinterpret_cast<uint32_t*>(a.ws + a.prefill_tickets);
        float* parts = reinterpret_cast<float*>(a.ws + a.prefill_parts);
        uint32_t ph_s = 0, ph_o = 0, ph_j = 0;
        auto half_barrier = [&]() {   // of the half's 128 threads, and bounded like every wait here
            mbar_arrive(joined(w));
            wait(joined(w), ph_j);
            ph_j ^= 1u;
        };
        // The row's Q of an item: f16, scaled, swizzled. Returns what turns its scores into powers of two. (The half's
        // products with the Q before it are done: their scores have been read.)
        auto load_q = [&](const PrefillItem& x) -> float {
            const int rows = x.rows - 128 * w;
            if (rows <= 0) return 0.0f;
            const int rr = x.first + 128 * w + min(row, rows - 1);
            const uint16_t* p = a.q + (long long)(x.row0 + rr / G) * a.q_stride + (long long)(x.h * G + rr % G) * D;
            uint4 v[D / 8];
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 8; i++) v[i] = row < rows ? *reinterpret_cast<const uint4*>(p + 8 * i) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < D / 8; i++) {
                const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int j = 0; j < 4; j++)
                    amax = max3(amax, fabsf(__uint_as_float(u[j] << 16)), fabsf(__uint_as_float(u[j] & 0xffff0000u)));
            }
            const int e = row_exponent(amax);
            const float down = pow2(-e);
#pragma unroll
            for (int i = 0; i < D / 8; i++) {
                const uint32_t u[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                uint32_t y[4];
#pragma unroll
                for (int j = 0; j < 4; j++)
                    y[j] = pack_f16(__uint_as_float(u[j] << 16) * down, __uint_as_float(u[j] & 0xffff0000u) * down);
                sts16(base + C::OFF_Q + (uint32_t)(w * C::PANELS + i / 8) * C::PANEL + (uint32_t)row * 128u +
                          (uint32_t)(((i & 7) ^ (row & 7)) << 4),
                      make_uint4(y[0], y[1], y[2], y[3]));
            }
            proxy_fence();
            mbar_arrive(q_full(w));
            return fmaxf(soft * pow2(e), 1e-37f);   // (a factor of 0 would turn masked scores into NaN)
        };
        const PrefillItem* item = take();
        float ksc_next = item != nullptr ? load_q(*item) : 0.0f;
        for (; item != nullptr; give_back()) {
            const PrefillItem& it = *item;
            const float ksc = ksc_next;
            const int rows = it.rows - 128 * w;   // of this half
            if (rows <= 0) {
                item = take(1);
                if (item != nullptr) ksc_next = load_q(*item);
                continue;
            }
            const int tile0 = it.tile0, qbase = it.kv_len - it.n;
            const int rr = it.first + 128 * w + min(row, rows - 1);
            const int tok_i = rr / G, head = it.h * G + rr % G;

            const int pos = qbase + tok_i;
            const int lim_hi = a.causal ? min(it.kv_len, pos + 1) : it.kv_len;
            const int lim_lo = a.window > 0 ? pos - a.window + 1 : 0;
            // between these every row of the half sees every token
            const int first_i = (it.first + 128 * w) / G, last_i = (it.first + 128 * w + min(rows, 128) - 1) / G;
            const int all_hi = a.causal ? min(it.kv_len, qbase + first_i + 1) : it.kv_len;
            const int all_lo = a.window > 0 ? qbase + last_i - a.window + 1 : 0;

            const int32_t* trow = a.table + (long long)it.b * a.cols;
            const int blk_hi = (it.hi + 15) >> 4;
            // Which of the next four tiles' 32 blocks lie in the cache: the ids are read four tiles ahead.
            auto page_id = [&](int k) {
                const int kb = (tile0 + k) * (PF_TILE / 16) + lane;
                return kb < blk_hi ? trow[kb >> page_shift] : -1;
            };
            int ids = page_id(it.k0);
            uint32_t there4 = 0;
            float m = NEG_BIG, l = 0.0f;
            for (int k = it.k0; k < it.k1; k++) {
                if (((k - it.k0) & 3) == 0) {
                    there4 = __ballot_sync(0xffffffffu, ids >= 0 && ids < a.cache.pages);
                    ids = page_id(k + 4);
                }
                const uint32_t there = there4 & 0xffu;
                there4 >>= 8;
                wait(s_full(w), ph_s);
                ph_s ^= 1u;
                tc_fence_after();
                const int tok = (tile0 + k) * PF_TILE;
                if (tok < all_lo || tok + PF_TILE > all_hi || there != 0xffu) {
                    // A tile with masked tokens: masked in place, in a loop of its own, so that the code that every
                    // tile runs through stays short (instruction fetch is what this loop waits for most).
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t s[32];
                        tc_ld32(ts + 32u * c, s);
                        tc_wait_ld_of(s);
                        const int lo = lim_lo - tok - c * 32, hi = lim_hi - tok - c * 32;
                        const uint32_t two = there >> (c * 2);
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (i < lo || i >= hi || !(two >> (i / 16) & 1u)) s[i] = __float_as_uint(-INFINITY);
                        tc_st32(ts + 32u * c, s);
                    }
                    tc_wait_st();
                }
                // Scores in four chunks of 32 columns: 0 and 1 are read for the maximum and once more for the
                // exponentials, 2 and 3 stay in registers in between. (All 128 at once spill, and with nearly
                // all of the L1 given to operands a spilled register comes back from L2.)
                auto max32 = [&](const uint32_t (&s)[32]) {
                    float u = __uint_as_float(s[0]), v = __uint_as_float(s[1]);
#pragma unroll
                    for (int i = 2; i < 30; i += 4) {
                        u = max3(u, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                        v = max3(v, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
                    }
                    return fmaxf(u, max3(v, __uint_as_float(s[30]), __uint_as_float(s[31])));
                };
                uint32_t x0[32], x1[32], x2[32];
                tc_ld32(ts, x0);
                tc_ld32(ts + 32u, x1);
                tc_ld32(ts + 64u, x2);
                tc_wait_ld_of(x0);
                tc_wait_ld_of(x1);
                tc_wait_ld_of(x2);
                float mx = fmaxf(max32(x0), max32(x1));
                tc_ld32(ts + 96u, x1);
                mx = fmaxf(mx, max32(x2));
                tc_wait_ld_of(x1);
                mx = fmaxf(mx, max32(x1));
                mx *= ksc;
                if (__any_sync(0xffffffffu, mx > m + 8.0f)) {
                    const float v = fmaxf(m, mx), f = exp2_approx(m - v);
                    m = v;
                    l *= f;
                    if (k > it.k0) {   // (the first tile's product overwrites O)
#pragma unroll 1
                        for (int c = 0; c < D / 32; c++) {
                            uint32_t o[32];
                            tc_ld32(to + 32u * c, o);
                            tc_wait_ld_of(o);
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tc_st32(to + 32u * c, o);
                        }
                    }
                }
                const float off = 6.0f - m;
                float l0 = 0.0f, l1 = 0.0f;
                // P over the second half of S: what a chunk's probabilities overwrite has been read. The product
                // over the last 64 tokens starts while the first are still being exponentiated.
                auto chunk = [&](const uint32_t (&s)[32], int c) {
                    uint32_t p[16];
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        float x = __uint_as_float(s[2 * i]), y = __uint_as_float(s[2 * i + 1]);
                        fma2(x, y, ksc, off);
                        x = exp2_approx(x);
                        y = exp2_approx(y);
                        add2(l0, l1, x, y);
                        p[i] = pack_f16(x, y);
                    }
                    tc_st16(ts + C::P_COL + 16u * c, p);
                };
#pragma unroll 1
                for (int c = 2; c >= 0; c -= 2) {
                    chunk(x2, c);
                    chunk(x1, c + 1);
                    if (c > 0) {
                        tc_ld32(ts, x2);
                        tc_ld32(ts + 32u, x1);
                        tc_wait_st();
                        tc_fence_before();
                        mbar_arrive(p_half(w));
                        tc_wait_ld_of(x2);
                        tc_wait_ld_of(x1);
                    }
                }
                l += l0 + l1;
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(p_full(w));
            }

            // The next item's Q before this one's result: its first products run meanwhile.
            item = take(1);
            if (item != nullptr) ksc_next = load_q(*item);

            // ---- result ----
            wait(o_full(w), ph_o);
            ph_o ^= 1u;
            tc_fence_after();
            const int c_first = it.c_first, c_begin = it.c_begin, c_end = it.c_end;
            const bool whole = c_begin == c_end;
            const int cta = blockIdx.x;
            uint16_t* dst = a.out + (long long)(it.row0 + tok_i) * a.out_stride + (long long)head * D;
            float* part = parts + (((long long)cta * 2 + (cta == c_first ? 1 : 0)) * 2 + w) * C::PART;
            const float inv = finish(1.0f, l, a.cache.v_div);
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                uint32_t o[32];
                tc_ld32(to + 32u * c, o);
                tc_wait_ld_of(o);
                if (whole) {
                    if (row < rows) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
                            *reinterpret_cast<uint4*>(dst + 32 * c + i) =
                                make_uint4(pack_bf16(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv),
                                           pack_bf16(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv),
                                           pack_bf16(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv),
                                           pack_bf16(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4*>(part + 256 + ((c * 8 + i / 4) * 128 + row) * 4) =
                            make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
            }
            tc_fence_before();
            mbar_arrive(o_empty(w));
            if (!whole) {
                part[row] = m;
                part[128 + row] = l;
                __threadfence();
                half_barrier();
                if (row == 0) s_last[w] = atomicAdd(&tickets[c_first * 2 + w], 1u) == (uint32_t)(c_end - c_begin);
                half_barrier();
                if (s_last[w]) {   // the half's last block: join the parts in token order
                    __threadfence();
                    if (row == 0) tickets[c_first * 2 + w] = 0;
                    auto part_of = [&](int c) { return parts + (((long long)c * 2 + (c == c_first ? 1 : 0)) * 2 + w) * C::PART; };
                    float mm = NEG_BIG, ll = 0.0f;
                    for (int c = c_begin; c <= c_end; c++) {
                        const float pm = __ldcg(part_of(c) + row), pl = __ldcg(part_of(c) + 128 + row), v = fmaxf(mm, pm);
                        ll = ll * exp2_approx(mm - v) + pl * exp2_approx(pm - v);
                        mm = v;
                    }
                    const float inv2 = finish(1.0f, ll, a.cache.v_div);
#pragma unroll 1
                    for (int d = 0; d < D; d += 64) {   // sixteen loads in flight per part
                        float o[64] = {};
#pragma unroll 1
                        for (int c = c_begin; c <= c_end; c++) {
                            const float* q = part_of(c);
                            float4 x[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) x[i] = __ldcg(reinterpret_cast<const float4*>(q + 256 + ((d / 4 + i) * 128 + row) * 4));
                            const float f = exp2_approx(__ldcg(q + row) - mm);
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                o[4 * i] += f * x[i].x;
                                o[4 * i + 1] += f * x[i].y;
                                o[4 * i + 2] += f * x[i].z;
                                o[4 * i + 3] += f * x[i].w;
                            }
                        }
                        if (row < rows) {
#pragma unroll
                            for (int i = 0; i < 64; i += 8)
                                *reinterpret_cast<uint4*>(dst + d + i) =
                                    make_uint4(pack_bf16(o[i] * inv2, o[i + 1] * inv2), pack_bf16(o[i + 2] * inv2, o[i + 3] * inv2),
                                               pack_bf16(o[i + 4] * inv2, o[i + 5] * inv2), pack_bf16(o[i + 6] * inv2, o[i + 7] * inv2));
                        }
                    }
                }
                half_barrier();   // (s_last)
            }
        }
    } else if (warp < 12) {
        // ---------------- 4-bit tiles to f16 operands ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 112;" ::: "memory");
        const int g = lane >> 2, t = lane & 3, wq = warp - 8;
        int n = 0;   // tiles so far: stage n & 1, its use n >> 1
        for (const PrefillItem* item; (item = take()) != nullptr; give_back()) {
            const PrefillItem& it = *item;
            const int tile0 = it.tile0, h = it.h, k_end = it.k1;
            const int32_t* trow = a.table + (long long)it.b * a.cols;
            const int blk_hi = (it.hi + 15) >> 4;
            auto page_of = [&](int k) {   // lane i: block i & 1 of this warp in tile k + i / 2
                const int kb = (tile0 + k + (lane >> 1)) * (PF_TILE / 16) + wq * 2 + (lane & 1);
                return kb < blk_hi && k + (lane >> 1) < k_end ? trow[kb >> page_shift] : -1;
            };
            auto block_at = [&](int id, int k, int which) -> const uint8_t* {
                if (id < 0 || id >= a.cache.pages) return nullptr;
                const int kb = (tile0 + k) * (PF_TILE / 16) + wq * 2 + which;
                return a.cache.blocks + ((((long long)id * hkv + h) << page_shift) + (kb & ((1 << page_shift) - 1))) * (18 * D);
            };
            int ids = page_of(it.k0), ids_at = it.k0;
            const uint8_t* blk[2];
            KRegs<D> kr[2];
            VRegs<D> vr[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                blk[i] = block_at(__shfl_sync(0xffffffffu, ids, i), it.k0, i);
                load_k<D>(kr[i], blk[i], lane);
            }
#pragma unroll
            for (int i = 0; i < 2; i++) load_v<D>(vr[i], blk[i], lane);
            for (int k = it.k0; k < k_end; k++, n++) {
                const int st = n & 1;
                const uint32_t ph = ((uint32_t)(n >> 1) & 1u) ^ 1u;
                wait(k_empty(st), ph);
                // K: lane (g, t) has tokens g and g + 8, dimensions t*D/4 ..: D/32 words of eight dimensions, one
                // 16-byte chunk each. In lanes t >= 2 the words are taken in another order (w ^ D/64), so that the
                // eight lanes of a store phase write eight different chunk positions.
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int hh = 0; hh < 2; hh++) {
                        const int tau = (wq * 2 + i) * 16 + hh * 8 + g;
                        const uint32_t rowp = base + C::OFF_K + (uint32_t)st * C::KV_BYTES + (uint32_t)tau * 128u;
                        const uint32_t b0 = (D == 128 ? kr[i].s >> (16 * hh) : kr[i].s >> (8 * hh)) & 0xffu;
                        const uint32_t b1 = D == 128 ? kr[i].s >> (16 * hh + 8) & 0xffu : b0;
                        const uint32_t sc[2] = {((b0 | b0 << 16) << 7) & 0x3f803f80u, ((b1 | b1 << 16) << 7) & 0x3f803f80u};
                        constexpr int W = D / 32;
                        const bool flip = t >= 2;
#pragma unroll
                        for (int x = 0; x < W; x++) {
                            const uint32_t word = flip ? kr[i].c[hh][x ^ (W / 2)] : kr[i].c[hh][x];
                            // (a scale covers 16 dimensions = two words)
                            const uint32_t s = W == 2 ? sc[0] : (flip ? sc[(x ^ (W / 2)) / 2] : sc[x / 2]);
                            uint32_t f[4];
                            codes_to_f16(word, f);
                            const int dim8 = t * W + (flip ? x ^ (W / 2) : x);   // eighth of the row
                            sts16(rowp + (uint32_t)(dim8 >> 3) * C::PANEL + (uint32_t)(((dim8 & 7) ^ (tau & 7)) << 4),
                                  make_uint4(mul_f16x2(f[0], s), mul_f16x2(f[1], s), mul_f16x2(f[2], s), mul_f16x2(f[3], s)));
                        }
                    }
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full(st));
                if (k + 1 < k_end) {
                    if (k + 1 - ids_at == 16) {
                        ids_at = k + 1;
                        ids = page_of(ids_at);
                    }
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        blk[i] = block_at(__shfl_sync(0xffffffffu, ids, (k + 1 - ids_at) * 2 + i), k + 1, i);
                        load_k<D>(kr[i], blk[i], lane);
                    }
                }
                wait(v_empty(st), ph);
                // V: lane (g, t) has tokens 8p + 2t + j, dimensions g*D/8 ..: D/64 chunks of eight dimensions per token;
                // chunk order flipped in odd lane groups (D = 128) for the same reason.
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int p = 0; p < 2; p++)
#pragma unroll
                        for (int j = 0; j < 2; j++) {
                            constexpr int W = D / 64;
                            const int tau = (wq * 2 + i) * 16 + p * 8 + 2 * t + j;
                            const uint32_t rowp = base + C::OFF_V + (uint32_t)st * C::KV_BYTES + (uint32_t)tau * 128u;
                            const uint32_t bs = vr[i].s >> (16 * p + 8 * j) & 0xffu;
                            const uint32_t s = ((bs | bs << 16) << 7) & 0x3f803f80u;
                            const bool flip = W == 2 && (g & 1);
#pragma unroll
                            for (int x = 0; x < W; x++) {
                                const uint32_t word = flip ? vr[i].c[p][j * W + (x ^ (W - 1))] : vr[i].c[p][j * W + x];
                                uint32_t f[4];
                                codes_to_f16(word, f);
                                const int dim8 = g * W + (flip ? x ^ (W - 1) : x);
                                sts16(rowp + (uint32_t)(dim8 >> 3) * C::PANEL + (uint32_t)(((dim8 & 7) ^ (tau & 7)) << 4),
                                      make_uint4(mul_f16x2(f[0], s), mul_f16x2(f[1], s), mul_f16x2(f[2], s), mul_f16x2(f[3], s)));
                            }
                        }
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full(st));
                if (k + 1 < k_end) {
#pragma unroll
                    for (int i = 0; i < 2; i++) load_v<D>(vr[i], blk[i], lane);
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;" ::: "memory");
        if (warp == 12) {
            // ---------------- MMA issue (the whole warp walks the loop, one lane issues) ----------------
            const bool leader = elect_one();
            const uint32_t idesc_s = f16_desc(128, false), idesc_o = f16_desc(D, true);
            int n = 0;
            uint32_t ph_q[2] = {0, 0}, ph_p[2] = {0, 0}, items[2] = {0, 0};
            auto product_s = [&](int w, int st) {
#pragma unroll
                for (int pd = 0; pd < C::PANELS; pd++) {
                    const uint64_t da = smem_desc_sw128(base + C::OFF_Q + (uint32_t)(w * C::PANELS + pd) * C::PANEL);
                    const uint64_t db = smem_desc_sw128(base + C::OFF_K + (uint32_t)st * C::KV_BYTES + (uint32_t)pd * C::PANEL);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        tc_mma<KIND_BF16, 1>(tmem + C::S_COL + 128u * w, da + 2u * j, db + 2u * j, idesc_s, pd + j > 0 ? 1u : 0u, 0, 0);
                }
            };
            auto product_o = [&](int w, int st, int j0, bool fresh) {
                const uint64_t db = smem_desc_v(base + C::OFF_V + (uint32_t)st * C::KV_BYTES, C::PANEL);
#pragma unroll
                for (int j = j0; j < j0 + 4; j++)   // sixteen tokens each
                    tc_mma_f16_ts(tmem + C::O_COL + (uint32_t)D * w, tmem + C::S_COL + C::P_COL + 128u * w + 8u * j, db + 128u * j, idesc_o,
                                  fresh && j == j0 ? 0u : 1u);
            };
            for (const PrefillItem* item; (item = take()) != nullptr; give_back()) {
                const PrefillItem& it = *item;
                const int halves = it.rows > 128 ? 2 : 1;
                const int count = it.k1 - it.k0;
                wait(k_full(n & 1), (uint32_t)(n >> 1) & 1u);
                for (int w = 0; w < halves; w++) {
                    wait(q_full(w), ph_q[w]);
                    ph_q[w] ^= 1u;
                    tc_fence_after();
                    if (leader) {
                        product_s(w, n & 1);
                        tc_commit(s_full(w));
                        if (w == halves - 1) tc_commit(k_empty(n & 1));
                    }
                }
                for (int i = 0; i < count; i++, n++) {
                    const int st = n & 1, nx = (n + 1) & 1;
                    const bool more = i + 1 < count;
                    wait(v_full(st), (uint32_t)(n >> 1) & 1u);
                    for (int w = 0; w < halves; w++) {
                        wait(p_half(w), ph_p[w]);
                        if (i == 0) {
                            wait(o_empty(w), (items[w] & 1u) ^ 1u);
                            items[w]++;
                        }
                        tc_fence_after();
                        if (leader) product_o(w, st, 4, i == 0);
                        if (w == 0 && more) wait(k_full(nx), (uint32_t)((n + 1) >> 1) & 1u);
                        wait(p_full(w), ph_p[w]);
                        ph_p[w] ^= 1u;
                        tc_fence_after();
                        if (leader) {
                            product_o(w, st, 0, false);
                            if (w == halves - 1) tc_commit(v_empty(st));
                            if (more) {
                                product_s(w, nx);
                                tc_commit(s_full(w));
                                if (w == halves - 1) tc_commit(k_empty(nx));
                            } else {
                                tc_commit(o_full(w));
                            }
                        }
                    }
                }
            }
            if (leader) tc_commit(drained);   // nothing of this block is in flight when tensor memory is freed
            wait(drained, 0);
        } else if (warp == 13) {
            // ---------------- the items, a few ahead ----------------
            Items<PF_ROWS, PF_TILE, PF_EXTRA> items(a, G, run, s_cut);
            for (int no = 0;; no++) {
                const int i = no % C::RING;
                wait(item_empty(i), ((uint32_t)(no / C::RING) & 1u) ^ 1u);
                const bool more = items.more() && !wait.given_up();
                if (lane == 0) {
                    PrefillItem x{};
                    if (more) {
                        x.k0 = items.k0;
                        x.k1 = items.k1;
                        x.tile0 = items.range.lo / PF_TILE;
                        x.hi = items.range.hi;
                        x.b = items.b;
                        x.h = items.h;
                        x.row0 = items.r.row0;
                        x.first = items.rt * PF_ROWS;
                        x.rows = min(PF_ROWS, items.r.n * G - x.first);
                        x.n = items.r.n;
                        x.kv_len = items.r.kv_len;
                        if (!items.whole()) {
                            const auto holders = items.holders();
                            x.c_first = holders.first;
                            x.c_begin = holders.begin;
                            x.c_end = holders.end;
                        }
                    }
                    s_items[i] = x;
                    mbar_arrive(item_full(i));
                }
                __syncwarp();
                if (!more) break;
                items.next(a, G);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

long long kv4_prefill_parts_bytes(int blocks, int head_dim) { return (long long)blocks * 4 * 128 * (head_dim + 2) * 4; }

template <int D>
static int launch_prefill(const Kv4AttnArgs& a, int blocks) {
    using C = PrefillCfg<D>;
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return VELOX_ERR_UNSUPPORTED;
    if (!ready[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kv4_prefill_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
        ready[dev] = true;
    }
    EarlyLaunch l((unsigned)blocks, PF_THREADS);
    l.cfg.dynamicSmemBytes = C::SMEM;
    cudaLaunchKernelEx(&l.cfg, kv4_prefill_kernel<D>, a);
    return launch_status();
}

int kv4_prefill(const Kv4AttnArgs& a, int blocks) {
    return a.cache.head_dim == 128 ? launch_prefill<128>(a, blocks) : launch_prefill<64>(a, blocks);
}

int kv4_status_sync() {
    int v = -1;
    if (cudaMemcpyFromSymbol(&v, g_kv4_status, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

int kv4_status_reset() {
    const int zero = 0;
    return (int)cudaMemcpyToSymbol(g_kv4_status, &zero, sizeof(int));
}

}  // namespace vx
