// Attention over the 4-bit key/value cache at decode widths: a few query rows per request and kv
// head against a long run of cached tokens.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,  j < kv_len, j <= pos_i (causal), j > pos_i - window
//
// The rows of one kv head (its group of query heads times the request's new tokens) share every
// byte of the cache, so they are the narrow side of the MMA: S^T = K Q^T with 16 tokens by 8 rows,
// then O^T = V^T P^T with 16 dimensions by 8 rows (mma.sync.m16n8k16). The accumulator layout of the first
// product becomes the operand layout of the second with one 8 x 8 transpose per eight tokens
// (movmatrix). Codes become f16 by the hardware conversion, times their scale: exact (six significant
// bits). q is scaled per row by a power of two into f16's range (exact but for values 2^-24 below the row's
// largest). P is rounded to f16 (2^-11; probabilities are scaled by 2^8 so that small ones stay
// normal), everything else is f32.
//
// Every warp streams its own blocks through a ring of its own in shared memory (cp.async, three steps of two
// blocks: up to 147 KB per SM on their way), so there is no barrier in the loop. The block layout (kv4.cuh) makes
// a lane's MMA operands one conflict-free access per plane. (Operands loaded straight into registers kept
// half as much in flight: 126 us against 109 us for 64 requests of 4k to 8k tokens, 64 / 8 heads of 128.)
// A block or page that is not there is read from the start of the cache instead (any byte is a finite
// number) and its scores are masked.
//
// Work is cut on the device (the lengths live there): all (request, kv head, row tile) items are laid
// end to end in units of one tile of tokens and every block takes an equal run, or, in short steps, an item or
// a part of one (kv4_items.cuh). A block that holds part of an item parks (max, sum, O) in the workspace, the last of the item's
// blocks to arrive joins them in token order: results do not depend on the order of arrival.
//
// What bounds it: issue. A block of 16 tokens (2304 bytes) takes 334 warp instructions, 196 of them the
// conversions, scalings and products of its 4096 values: 64 requests of 8192 tokens stream at 4.8 TB/s (73 % of a
// copy; the slope between 428 and 604 MB is 6.6 TB/s), the rest is 8 us from launch to first bytes and 2 to 3 us per item.
#include "common.cuh"
#include "kv4.cuh"
#include "kv4_items.cuh"

namespace vx {

__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    const __nv_bfloat162 v = __float22bfloat162_rn(make_float2(lo, hi));
    return *reinterpret_cast<const uint32_t*>(&v);
}

constexpr int DECODE_EXTRA = 1;   // tiles' worth of an item's other costs
constexpr int DECODE_JOIN = 3;    // and of joining its parts

template <int D, int NT, int WARPS>
struct DecodeCfg {
    static constexpr int ROWS = 8 * NT;            // query rows of an item
    static constexpr int STEP = 32;                // tokens per warp and step: two blocks
    static constexpr int TILE = WARPS * STEP;      // tokens per unit of work
    static constexpr int THREADS = WARPS * 32;
    static constexpr int STRIDE = D + 4;           // padded f32 row in shared memory
    static constexpr int BLOCK = 18 * D, STAGE = 2 * BLOCK, STAGES = 3;
    static constexpr int RING = WARPS * STAGES * STAGE;
    static constexpr int JOIN = WARPS * ROWS * STRIDE * 4 + 2 * WARPS * ROWS * 4;   // over the ring
    static constexpr int SMEM = RING > JOIN ? RING : JOIN;
    // a parked part: max, sum per row, then O
    static constexpr int PART = ROWS * (D + 2);
};

// (Offsets are immediates of the instructions: an address each in registers was a quarter of the loop's
// instructions, and the loop is bound by their issue.)
template <int OFF>
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0 + %2], [%1 + %2], 16;" ::"r"(dst), "l"(src), "n"(OFF) : "memory");
}
// The two blocks of a step into a stage, by the whole warp: 2 * 18 D bytes, lane by lane in 16-byte chunks.
template <int D, int I = 0>
__device__ __forceinline__ void copy_step(uint32_t dst, const uint8_t* p0, const uint8_t* p1, int lane) {
    // dst, p0: at the lane's first chunk; p1: as if its block followed p0's
    constexpr int CHUNKS = 18 * D / 16, ALL = 2 * CHUNKS;   // 144 or 72 per block
    if constexpr (32 * I < ALL) {
        constexpr bool first = 32 * I + 31 < CHUNKS, both = 32 * I < CHUNKS && !first;
        const uint8_t* src = first || (both && lane < CHUNKS - 32 * I) ? p0 : p1;
        if (32 * I + 31 < ALL || lane < ALL - 32 * I) copy16<512 * I>(dst, src);
        copy_step<D, I + 1>(dst, p0, p1, lane);
    }
}
// A lane's operands of a block in shared memory.
template <int D, int OFF>
__device__ __forceinline__ void lds_plane(uint32_t (&c)[2][D / 32], uint32_t lane_piece) {
    if constexpr (D == 128) {
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
                     : "=r"(c[0][0]), "=r"(c[0][1]), "=r"(c[0][2]), "=r"(c[0][3]) : "r"(lane_piece), "n"(OFF));
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
                     : "=r"(c[1][0]), "=r"(c[1][1]), "=r"(c[1][2]), "=r"(c[1][3]) : "r"(lane_piece), "n"(OFF + 512));
    } else {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(c[0][0]), "=r"(c[0][1]) : "r"(lane_piece), "n"(OFF));
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(c[1][0]), "=r"(c[1][1]) : "r"(lane_piece), "n"(OFF + 256));
    }
}
// piece: the stage plus the lane's place in a code plane; k_scale, v_scale: plus its place in a scale plane.
template <int D, int OFF>
__device__ __forceinline__ void lds_k(KRegs<D>& r, uint32_t piece, uint32_t k_scale) {
    lds_plane<D, OFF>(r.c, piece);
    if constexpr (D == 128) {
        asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(r.s) : "r"(k_scale), "n"(OFF + 16 * D));
    } else {
        uint16_t v;
        asm volatile("ld.shared.u16 %0, [%1 + %2];" : "=h"(v) : "r"(k_scale), "n"(OFF + 16 * D));
        r.s = v;
    }
}
template <int D, int OFF>
__device__ __forceinline__ void lds_v(VRegs<D>& r, uint32_t piece, uint32_t v_scale) {
    lds_plane<D, OFF + 8 * D>(r.c, piece);
    asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(r.s) : "r"(v_scale), "n"(OFF + 17 * D));
}

// S^T of one block of 16 tokens: c[n] rows g, g + 8 = tokens, columns 2t, 2t + 1 of row tile n.
template <int D, int NT>
__device__ __forceinline__ void scores(const KRegs<D>& k, const uint32_t (&qf)[NT][D / 16][2], float (&c)[NT][4]) {
#pragma unroll
    for (int n = 0; n < NT; n++) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f;
    uint32_t s0[D / 64], s1[D / 64];
    if (D == 128) {
        s0[0] = scale_pair(k.s, 0x4040); s0[D / 64 - 1] = scale_pair(k.s, 0x4141);
        s1[0] = scale_pair(k.s, 0x4242); s1[D / 64 - 1] = scale_pair(k.s, 0x4343);
    } else {
        s0[0] = scale_pair(k.s, 0x4040);
        s1[0] = scale_pair(k.s, 0x4141);
    }
#pragma unroll
    for (int w = 0; w < D / 32; w++) {
        uint32_t x[4], y[4];
        codes_to_f16(k.c[0][w], x);
        codes_to_f16(k.c[1][w], y);
        const uint32_t sx = s0[w / 2], sy = s1[w / 2];   // 16 dimensions = two words
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t a0 = mul_f16x2(x[2 * j], sx), a1 = mul_f16x2(y[2 * j], sy);
            const uint32_t a2 = mul_f16x2(x[2 * j + 1], sx), a3 = mul_f16x2(y[2 * j + 1], sy);
#pragma unroll
            for (int n = 0; n < NT; n++) mma16816(c[n], a0, a1, a2, a3, qf[n][2 * w + j][0], qf[n][2 * w + j][1]);
        }
    }
}

// O^T += V^T P^T of one block: o[n][i] rows g, g + 8 = dimensions 2i, 2i + 1 of lane group g's D/8.
template <int D, int NT>
__device__ __forceinline__ void accumulate(const VRegs<D>& v, const uint32_t (&p)[NT][2], float (&o)[NT][D / 16][4]) {
    const uint32_t sa = scale_pair(v.s, 0x4140), sb = scale_pair(v.s, 0x4342);
    constexpr int W = D / 64;   // words per piece
#pragma unroll
    for (int w = 0; w < W; w++) {
        uint32_t al[4], ah[4], bl[4], bh[4];
        {
            const uint32_t x = v.c[0][w], y = v.c[0][W + w];
            codes_to_f16((x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u), al);
            codes_to_f16(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), ah);
        }
        {
            const uint32_t x = v.c[1][w], y = v.c[1][W + w];
            codes_to_f16((x & 0x0f0f0f0fu) | ((y << 4) & 0xf0f0f0f0u), bl);
            codes_to_f16(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u), bh);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t a0 = mul_f16x2(al[j], sa), a1 = mul_f16x2(ah[j], sa);
            const uint32_t a2 = mul_f16x2(bl[j], sb), a3 = mul_f16x2(bh[j], sb);
#pragma unroll
            for (int n = 0; n < NT; n++) mma16816(o[n][w * 4 + j], a0, a1, a2, a3, p[n][0], p[n][1]);
        }
    }
}

template <int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 2 : 1)
kv4_decode_kernel(const __grid_constant__ Kv4AttnArgs a) {
    using C = DecodeCfg<D, NT, WARPS>;
    constexpr int ROWS = C::ROWS, TILE = C::TILE;
    // (128: copies into rows of it that straddle lines cost 8 % at long lengths)
    extern __shared__ __align__(128) float smem[];
    float* s_o = smem;                                   // [WARPS][ROWS][STRIDE]
    float* s_m = smem + WARPS * ROWS * C::STRIDE;        // [WARPS][ROWS] max, then sum
    __shared__ long long s_red[WARPS], s_found[2];
    __shared__ int s_last;
    __shared__ Cut s_cut;
    __shared__ float s_sum[ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int hkv = a.cache.kv_heads, G = a.heads / hkv, page_shift = a.cache.page_shift - 4;   // of blocks per page
    if (tid == 0) grid_launch_dependents();
    grid_dependency_wait();

    const Run run = find_run<ROWS, TILE, DECODE_EXTRA, C::THREADS, 4, DECODE_JOIN>(a, G, s_red, s_cut, s_found);
    if ((int)blockIdx.x >= run.blocks) return;
    const float soft = score_factor(a);
    uint32_t* tickets = reinterpret_cast<uint32_t*>(a.ws);
    float* parts = reinterpret_cast<float*>(a.ws + a.decode_parts);

    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + (tid >> 5) * (C::STAGES * C::STAGE);
    Items<ROWS, TILE, DECODE_EXTRA> it(a, G, run, s_cut);
    for (; it.more(); it.next(a, G)) {
        const Request& r = it.r;
        const RowRange range = it.range;
        const int b = it.b, h = it.h, rt = it.rt, k0 = it.k0, k1 = it.k1;
        const int tile0 = range.lo / TILE;
        const int rows = min(ROWS, r.n * G - rt * ROWS);
        const int qbase = r.kv_len - r.n;

        // Page ids of this warp's next sixteen steps, and of the sixteen after them: lane i holds the id of block
        // i & 1 of step i / 2.
        const int32_t* trow = a.table + (long long)b * a.cols;
        const int blk_hi = (range.hi + 15) >> 4;
        const int kb0 = tile0 * (TILE / 16) + warp * 2;   // first block of step 0
        auto page_of = [&](int k) {
            const int kb = kb0 + (k + (lane >> 1)) * (TILE / 16) + (lane & 1);
            return kb < blk_hi && k + (lane >> 1) < k1 ? trow[kb >> page_shift] : -1;
        };
        int ids = page_of(k0), ids_next = page_of(k0 + 16);

        // ---- the rows' operands and limits ----
        uint32_t qf[NT][D / 16][2];
        float ksc[NT][2];
        int lim_lo[NT][2], lim_hi[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int row = n * 8 + g;
            float x[D / 4];
            if (row < rows) {
                const int rr = rt * ROWS + row;
                const uint16_t* p = a.q + (long long)(r.row0 + rr / G) * a.q_stride + (long long)(h * G + rr % G) * D + t * (D / 4);
#pragma unroll
                for (int i = 0; i < D / 32; i++) {
                    const uint4 w = *reinterpret_cast<const uint4*>(p + 8 * i);
                    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        x[8 * i + 2 * j] = __uint_as_float(ww[j] << 16);
                        x[8 * i + 2 * j + 1] = __uint_as_float(ww[j] & 0xffff0000u);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < D / 4; i++) x[i] = 0.0f;
            }
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 4; i++) amax = fmaxf(amax, fabsf(x[i]));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int e = row_exponent(amax);
            const float down = pow2(-e);
#pragma unroll
            for (int j = 0; j < D / 16; j++) {
                qf[n][j][0] = pack_f16(x[4 * j] * down, x[4 * j + 1] * down);
                qf[n][j][1] = pack_f16(x[4 * j + 2] * down, x[4 * j + 3] * down);
            }
            const float up = fmaxf(soft * pow2(e), 1e-37f);   // (a factor of 0 would turn masked scores into NaN)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int col = n * 8 + 2 * t + c;
                ksc[n][c] = __shfl_sync(0xffffffffu, up, (2 * t + c) * 4);
                const int pos = qbase + (rt * ROWS + min(col, rows - 1)) / G;
                lim_hi[n][c] = a.causal ? min(r.kv_len, pos + 1) : r.kv_len;
                lim_lo[n][c] = a.window > 0 ? pos - a.window + 1 : 0;
            }
        }
        // between these every row sees every token
        const int all_hi = a.causal ? min(r.kv_len, qbase + rt * ROWS / G + 1) : r.kv_len;
        const int all_lo = a.window > 0 ? qbase + (rt * ROWS + rows - 1) / G - a.window + 1 : 0;

        float m[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            m[n][0] = m[n][1] = NEG_BIG;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 16; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
        }

        const uint8_t* head = a.cache.blocks + ((long long)h << page_shift) * C::BLOCK + lane * 16;
        const uint32_t page_bytes = ((uint32_t)hkv << page_shift) * C::BLOCK, page_mask = (1u << page_shift) - 1;
        uint32_t have = 0;        // two bits per step on its way, the oldest lowest
        int issued = k0;
        uint32_t in = ring + lane * 16;
        __syncthreads();          // (the ring is the join's memory of the item before)
        auto issue = [&](int ahead) {   // the step `ahead` of the one that is read next
            if (issued < k1) {
                const int at = (issued - k0) & 15;
                if (at == 0 && issued != k0) {
                    ids = ids_next;
                    ids_next = page_of(issued + 16);
                }
                const uint32_t kb = kb0 + issued * (TILE / 16);
                uint32_t id = __shfl_sync(0xffffffffu, ids, at * 2);
                uint32_t bits = id < (uint32_t)a.cache.pages ? 3u : 0u;
                const uint8_t* p0 = head + (unsigned long long)(bits ? id : 0u) * page_bytes + (kb & page_mask) * C::BLOCK;
                const uint8_t* p1 = p0;   // pages of 32 tokens and more: the step's second block follows its first
                if (page_shift == 0) {
                    id = __shfl_sync(0xffffffffu, ids, at * 2 + 1);
                    const bool there = id < (uint32_t)a.cache.pages;
                    bits = (bits & 1u) | (there ? 2u : 0u);
                    p1 = head + (unsigned long long)(there ? id : 0u) * page_bytes - C::BLOCK;
                }
                have |= bits << (2 * ahead);
                copy_step<D>(in, p0, p1, lane);
                in = in == ring + lane * 16 + (C::STAGES - 1) * C::STAGE ? ring + lane * 16 : in + C::STAGE;
            }
            issued++;
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < C::STAGES - 1; i++) issue(i);

        int slot = 0;
        for (int k = k0; k < k1; k++) {
            issue(C::STAGES - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(C::STAGES - 1) : "memory");
            __syncwarp();
            const uint32_t stage = ring + slot * C::STAGE;
            slot = slot == C::STAGES - 1 ? 0 : slot + 1;
            const uint32_t there = have & 3u;
            have >>= 2;
            const uint32_t piece = stage + lane * (D / 8), k_scale = stage + lane * (D / 32);
            const uint32_t v_scale = stage + (D == 128 ? lane : (lane >> 3) * 4 + (lane & 3)) * 4;
            float c[2][NT][4];
            {
                KRegs<D> kr;
                lds_k<D, 0>(kr, piece, k_scale);
                scores<D, NT>(kr, qf, c[0]);
                lds_k<D, C::BLOCK>(kr, piece, k_scale);
                scores<D, NT>(kr, qf, c[1]);
            }
            const int tok = (tile0 + k) * TILE + warp * 32;
            if (tok < all_lo || tok + 32 > all_hi || there != 3u) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const int j = tok + i * 16 + g + (x >> 1) * 8;
                            if (j < lim_lo[n][x & 1] || j >= lim_hi[n][x & 1] || !(there >> i & 1u)) c[i][n][x] = -INFINITY;
                        }
            }
            // running maximum of each row (column of S^T), over the lanes that share the column
            uint32_t pf[2][NT][2];
            bool grew = false;
            float mx[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const float v = fmaxf(fmaxf(c[0][n][y], c[0][n][y + 2]), fmaxf(c[1][n][y], c[1][n][y + 2]));
                    mx[n][y] = v * ksc[n][y];
                    grew = grew || mx[n][y] > m[n][y];
                }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        float v = fmaxf(m[n][y], mx[n][y]);
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
                        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
                        const float f = exp2_approx(m[n][y] - v);
                        m[n][y] = v;
                        l[n][y] *= f;
#pragma unroll
                        for (int i = 0; i < D / 16; i++) {
                            o[n][i][y] *= f;
                            o[n][i][y + 2] *= f;
                        }
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float off[2] = {8.0f - m[n][0], 8.0f - m[n][1]};
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float p[4];
#pragma unroll
                    for (int x = 0; x < 4; x++) p[x] = exp2_approx(fmaf(c[i][n][x], ksc[n][x & 1], off[x & 1]));
                    l[n][0] += p[0] + p[2];
                    l[n][1] += p[1] + p[3];
                    pf[i][n][0] = transpose8x8(pack_f16(p[0], p[1]));
                    pf[i][n][1] = transpose8x8(pack_f16(p[2], p[3]));
                }
            }
            {
                VRegs<D> vr;
                lds_v<D, 0>(vr, piece, v_scale);
                accumulate<D, NT>(vr, pf[0], o);
                lds_v<D, C::BLOCK>(vr, piece, v_scale);
                accumulate<D, NT>(vr, pf[1], o);
            }
            __syncwarp();   // before the stage is written again
        }
        asm volatile("cp.async.wait_all;" ::: "memory");

        // ---- join the warps ----
        // Rows are kept in the order [i][g][2]: dimension g * D/8 + 2i + e at i * 16 + 2g + e; a thread joins four
        // neighbours of it.
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float sum = l[n][y];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int row = n * 8 + 2 * t + y;
                if (g == 0) {
                    s_m[warp * ROWS + row] = m[n][y];
                    s_m[(WARPS + warp) * ROWS + row] = sum;
                }
#pragma unroll
                for (int i = 0; i < D / 16; i++)
                    *reinterpret_cast<float2*>(s_o + (warp * ROWS + row) * C::STRIDE + i * 16 + 2 * g) =
                        make_float2(o[n][i][y], o[n][i][y + 2]);
            }
        const bool whole = it.whole();
        int c_first = 0, c_begin = 0, count = 1;
        if (!whole) {
            const auto holders = it.holders();
            c_first = holders.first;
            c_begin = holders.begin;
            count = holders.end - c_begin + 1;
        }
        float* part = parts + ((long long)blockIdx.x * 2 + ((int)blockIdx.x == c_first ? 1 : 0)) * C::PART;
        __syncthreads();
        if (tid < ROWS) {   // the warps' factors, and the row's maximum and sum
            float mm = NEG_BIG, ll = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) mm = fmaxf(mm, s_m[w * ROWS + tid]);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float f = exp2_approx(s_m[w * ROWS + tid] - mm);
                ll += f * s_m[(WARPS + w) * ROWS + tid];
                s_m[w * ROWS + tid] = f;
            }
            s_sum[tid] = finish(1.0f, ll, a.cache.v_div);
            if (!whole) {
                part[tid] = mm;
                part[ROWS + tid] = ll;
            }
        }
        __syncthreads();
        auto write = [&](int row, int at, const float4& v, float inv) {   // four results of a row that exists
            const int rr = rt * ROWS + row, d = (at & 15) / 2 * (D / 8) + at / 16 * 2;
            uint16_t* dst = a.out + (long long)(r.row0 + rr / G) * a.out_stride + (long long)(h * G + rr % G) * D + d;
            *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(v.x * inv, v.y * inv);
            *reinterpret_cast<uint32_t*>(dst + D / 8) = pack_bf16x2(v.z * inv, v.w * inv);
        };
        for (int i = tid; i < ROWS * D / 4; i += C::THREADS) {
            const int row = i / (D / 4), at = i % (D / 4) * 4;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float f = s_m[w * ROWS + row];
                const float4 v = *reinterpret_cast<const float4*>(s_o + (w * ROWS + row) * C::STRIDE + at);
                acc.x += f * v.x;
                acc.y += f * v.y;
                acc.z += f * v.z;
                acc.w += f * v.w;
            }
            if (!whole)
                *reinterpret_cast<float4*>(part + 2 * ROWS + row * D + at) = acc;
            else if (row < rows)
                write(row, at, acc, s_sum[row]);
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicAdd(&tickets[c_first], 1u) == (uint32_t)(count - 1);
            __syncthreads();
            if (s_last) {   // the item's last block: join the parts in token order
                __threadfence();
                if (tid == 0) tickets[c_first] = 0;
                auto part_of = [&](int c) { return parts + ((long long)(c_begin + c) * 2 + (c_begin + c == c_first ? 1 : 0)) * C::PART; };
                float* s_f = smem;                      // [count][ROWS]: maxima, then factors
                float* s_l = smem + count * ROWS;       // sums
                for (int i = tid; i < count * ROWS; i += C::THREADS) {
                    s_f[i] = __ldcg(part_of(i / ROWS) + i % ROWS);
                    s_l[i] = __ldcg(part_of(i / ROWS) + ROWS + i % ROWS);
                }
                __syncthreads();
                for (int row = warp; row < ROWS; row += WARPS) {
                    float mm = NEG_BIG, ll = 0.0f;
                    for (int c = lane; c < count; c += 32) mm = fmaxf(mm, s_f[c * ROWS + row]);
                    mm = warp_max(mm);
                    for (int c = lane; c < count; c += 32) {
                        const float f = exp2_approx(s_f[c * ROWS + row] - mm);
                        ll += f * s_l[c * ROWS + row];
                        s_f[c * ROWS + row] = f;
                    }
                    ll = warp_sum(ll);
                    if (lane == 0) s_sum[row] = finish(1.0f, ll, a.cache.v_div);
                }
                __syncthreads();
                for (int i = tid; i < rows * D / 4; i += C::THREADS) {
                    const int row = i / (D / 4), at = i % (D / 4) * 4;
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                    for (int c = 0; c < count; c++) {
                        const float f = s_f[c * ROWS + row];
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(part_of(c) + 2 * ROWS + row * D + at));
                        acc.x += f * v.x;
                        acc.y += f * v.y;
                        acc.z += f * v.z;
                        acc.w += f * v.w;
                    }
                    write(row, at, acc, s_sum[row]);
                }
            }
        }
    }
}

static int attn_sms() {
    static int sms[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (sms[dev] == 0) {
        int n = 0;
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
        sms[dev] = n > 0 ? n : 148;
    }
    return sms[dev];
}

constexpr int DECODE_WARPS = 8, DECODE_PER_SM = 2;
// Query rows per kv head and request up to which the decode kernel takes a request.
constexpr int DECODE_ROWS = 32;

// [decode tickets][prefill tickets][decode parts][prefill parts]; the tickets are zero between calls
struct WsLayout {
    int decode_blocks, prefill_blocks;
    long long prefill_tickets, decode_parts, prefill_parts, bytes;
};
static WsLayout ws_layout(int head_dim) {
    WsLayout w;
    w.prefill_blocks = attn_sms();
    w.decode_blocks = DECODE_PER_SM * attn_sms();
    auto up = [](long long x) { return (x + 255) & ~255LL; };
    w.prefill_tickets = up(4LL * w.decode_blocks);
    w.decode_parts = up(w.prefill_tickets + 8LL * w.prefill_blocks);
    w.prefill_parts = up(w.decode_parts + (long long)w.decode_blocks * 2 * 16 * (head_dim + 2) * 4);
    w.bytes = w.prefill_parts + kv4_prefill_parts_bytes(w.prefill_blocks, head_dim);
    return w;
}

long long kv4_attention_workspace(int head_dim) { return ws_layout(head_dim).bytes; }

template <int D, int NT>
static int launch_decode(const Kv4AttnArgs& a, int blocks) {
    using C = DecodeCfg<D, NT, DECODE_WARPS>;
    auto kern = kv4_decode_kernel<D, NT, DECODE_WARPS>;
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return VELOX_ERR_UNSUPPORTED;
    if (!ready[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
        ready[dev] = true;
    }
    EarlyLaunch l((unsigned)blocks, C::THREADS);
    l.cfg.dynamicSmemBytes = C::SMEM;
    cudaLaunchKernelEx(&l.cfg, kern, a);
    return launch_status();
}

int kv4_attention(Kv4AttnArgs a) {
    const WsLayout w = ws_layout(a.cache.head_dim);
    a.prefill_tickets = w.prefill_tickets;
    a.decode_parts = w.decode_parts;
    a.prefill_parts = w.prefill_parts;
    const int G = a.heads / a.cache.kv_heads;
    const long long most = (long long)a.max_new * G;
    // Two kernels share a call whose requests may be of both kinds; each passes over the other's. (The
    // lengths are on the device, so the host goes by max_new alone.)
    if (G <= DECODE_ROWS) {
        a.min_rows = 0;
        a.max_rows = DECODE_ROWS;
        int rc;
        if (a.cache.head_dim == 128)
            rc = most <= 8 ? launch_decode<128, 1>(a, w.decode_blocks) : launch_decode<128, 2>(a, w.decode_blocks);
        else
            rc = most <= 8 ? launch_decode<64, 1>(a, w.decode_blocks) : launch_decode<64, 2>(a, w.decode_blocks);
        if (rc != 0 || most <= DECODE_ROWS) return rc;
    }
    a.min_rows = G <= DECODE_ROWS ? DECODE_ROWS : 0;
    a.max_rows = 0x7fffffff;
    return kv4_prefill(a, w.prefill_blocks);
}

}  // namespace vx
