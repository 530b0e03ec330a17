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
// Bytes reach the warps as MMA operands straight from global memory (the cache's block layout, kv4.cuh):
// no shared memory, no barrier in the loop. The blocks of a step are requested as soon as the
// registers that hold the step before are free, K during the softmax and V product, V during the
// next K product.
//
// Work is cut by length, on the device (the lengths live there): all (request, kv head, row tile)
// items are laid end to end in units of one tile of tokens, every block takes an equal run. A
// block that holds part of an item parks (max, sum, O) in the workspace, the last of the item's
// blocks to arrive joins them in token order: results do not depend on the order of arrival.
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
template <int D, int NT, int WARPS>
struct DecodeCfg {
    static constexpr int ROWS = 8 * NT;            // query rows of an item
    static constexpr int STEP = 32;                // tokens per warp and step: two blocks
    static constexpr int TILE = WARPS * STEP;      // tokens per unit of work
    static constexpr int THREADS = WARPS * 32;
    static constexpr int STRIDE = D + 4;           // padded f32 row in shared memory
    static constexpr int SMEM = WARPS * ROWS * STRIDE * 4 + 2 * WARPS * ROWS * 4;
    // a parked part: max, sum per row, then O
    static constexpr int PART = ROWS * (D + 2);
};

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
    extern __shared__ float smem[];
    float* s_o = smem;                                   // [WARPS][ROWS][STRIDE]
    float* s_m = smem + WARPS * ROWS * C::STRIDE;        // [WARPS][ROWS] max, then sum
    __shared__ long long s_red[WARPS], s_found[2];
    __shared__ int s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int hkv = a.cache.kv_heads, G = a.heads / hkv, page_shift = __ffs(a.cache.page_size) - 5;   // (blocks per page: a power of two)
    if (tid == 0) grid_launch_dependents();
    grid_dependency_wait();

    const Run run = find_run<ROWS, TILE, C::THREADS>(a, G, s_red, s_found);
    if ((int)blockIdx.x >= run.blocks) return;
    const int cta = blockIdx.x;
    const float soft = score_factor(a);
    uint32_t* tickets = reinterpret_cast<uint32_t*>(a.ws);
    float* parts = reinterpret_cast<float*>(a.ws + a.decode_parts);

    Items<ROWS, TILE> it(a, G, run);
    for (; it.more(); it.next(a, G)) {
        const Request& r = it.r;
        const RowRange range = it.range;
        const int b = it.b, h = it.h, rt = it.rt, k0 = it.k0, k1 = it.k1;
        const int tile0 = range.lo / TILE;
        const int rows = min(ROWS, r.n * G - rt * ROWS);
        const int qbase = r.kv_len - r.n;

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
            const float up = soft * pow2(e);
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

        // Page ids of this warp's next sixteen steps: lane i holds the id of block i & 1 of step i / 2.
        const int32_t* trow = a.table + (long long)b * a.cols;
        const int blk_hi = (range.hi + 15) >> 4;
        auto page_of = [&](int k) {
            const int kb = (tile0 + k + (lane >> 1)) * (TILE / 16) + warp * 2 + (lane & 1);
            return kb < blk_hi ? trow[kb >> page_shift] : -1;
        };
        auto block_at = [&](int id, int k, int which) -> const uint8_t* {
            if (id < 0 || id >= a.cache.pages) return nullptr;
            const int kb = (tile0 + k) * (TILE / 16) + warp * 2 + which;
            return a.cache.blocks + ((((long long)id * hkv + h) << page_shift) + (kb & ((1 << page_shift) - 1))) * (18 * D);
        };
        int ids = page_of(k0), ids_at = k0;
        const uint8_t* blk[2];
        KRegs<D> kr[2];
        VRegs<D> vr[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            blk[i] = block_at(__shfl_sync(0xffffffffu, ids, i), k0, i);
            load_k<D>(kr[i], blk[i], lane);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) load_v<D>(vr[i], blk[i], lane);

        for (int k = k0; k < k1; k++) {
            float c[2][NT][4];
            const bool have0 = blk[0] != nullptr, have1 = blk[1] != nullptr;
#pragma unroll
            for (int i = 0; i < 2; i++) scores<D, NT>(kr[i], qf, c[i]);
            if (k + 1 < k1) {   // K of the next step
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
            const int tok = (tile0 + k) * TILE + warp * 32;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int x = 0; x < 4; x++) c[i][n][x] *= ksc[n][x & 1];
            if (tok < all_lo || tok + 32 > all_hi || !have0 || !have1) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const int j = tok + i * 16 + g + (x >> 1) * 8;
                            if (j < lim_lo[n][x & 1] || j >= lim_hi[n][x & 1] || !(i == 0 ? have0 : have1))
                                c[i][n][x] = -INFINITY;
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
                    float v = fmaxf(fmaxf(c[0][n][y], c[0][n][y + 2]), fmaxf(c[1][n][y], c[1][n][y + 2]));
                    grew = grew || v > m[n][y];
                    mx[n][y] = v;
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
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float p[4];
#pragma unroll
                    for (int x = 0; x < 4; x++) p[x] = exp2_approx(c[i][n][x] - m[n][x & 1] + 8.0f);
                    l[n][0] += p[0] + p[2];
                    l[n][1] += p[1] + p[3];
                    pf[i][n][0] = transpose8x8(pack_f16(p[0], p[1]));
                    pf[i][n][1] = transpose8x8(pack_f16(p[2], p[3]));
                }
#pragma unroll
            for (int i = 0; i < 2; i++) accumulate<D, NT>(vr[i], pf[i], o);
            if (k + 1 < k1) {
#pragma unroll
                for (int i = 0; i < 2; i++) load_v<D>(vr[i], blk[i], lane);
            }
        }

        // ---- join the warps ----
        __syncthreads();   // (shared memory of the item before)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float s = l[n][y];
                s += __shfl_xor_sync(0xffffffffu, s, 4);
                s += __shfl_xor_sync(0xffffffffu, s, 8);
                s += __shfl_xor_sync(0xffffffffu, s, 16);
                const int row = n * 8 + 2 * t + y;
                if (g == 0) {
                    s_m[warp * ROWS + row] = m[n][y];
                    s_m[(WARPS + warp) * ROWS + row] = s;
                }
            }
        // rows in the order [i][g][2]: dimension g * D/8 + 2i + e at i * 16 + 2g + e
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int y = 0; y < 2; y++)
                    *reinterpret_cast<float2*>(s_o + (warp * ROWS + n * 8 + 2 * t + y) * C::STRIDE + i * 16 + 2 * g) =
                        make_float2(o[n][i][y], o[n][i][y + 2]);
        __syncthreads();
        const bool whole = it.whole();
        const int c_first = it.first_block(), c_last = it.last_block();
        float* part = parts + ((long long)cta * 2 + (cta == c_first ? 1 : 0)) * C::PART;
        for (int i = tid; i < ROWS * D; i += C::THREADS) {
            const int row = i / D, d = i % D;
            const int at = (d % (D / 8)) / 2 * 16 + d / (D / 8) * 2 + (d & 1);
            float mm = NEG_BIG;
#pragma unroll
            for (int w = 0; w < WARPS; w++) mm = fmaxf(mm, s_m[w * ROWS + row]);
            float acc = 0.0f, ll = 0.0f;
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                const float f = exp2_approx(s_m[w * ROWS + row] - mm);
                acc += f * s_o[(w * ROWS + row) * C::STRIDE + at];
                ll += f * s_m[(WARPS + w) * ROWS + row];
            }
            if (whole) {
                if (row < rows) {
                    const int rr = rt * ROWS + row;
                    a.out[(long long)(r.row0 + rr / G) * a.out_stride + (long long)(h * G + rr % G) * D + d] =
                        bf16_bits(finish(acc, ll, a.cache.v_div));
                }
            } else {
                part[2 * ROWS + i] = acc;
                if (d == 0) {
                    part[row] = mm;
                    part[ROWS + row] = ll;
                }
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicAdd(&tickets[c_first], 1u) == (uint32_t)(c_last - c_first);
            __syncthreads();
            if (s_last) {   // the item's last block: join the parts in token order
                __threadfence();
                if (tid == 0) tickets[c_first] = 0;
                for (int i = tid; i < rows * D; i += C::THREADS) {
                    const int row = i / D, d = i % D;
                    float mm = NEG_BIG, acc = 0.0f, ll = 0.0f;
                    for (int c = c_first; c <= c_last; c++) {
                        const float* q = parts + ((long long)c * 2 + (c == c_first ? 1 : 0)) * C::PART;
                        const float pm = __ldcg(q + row), pl = __ldcg(q + ROWS + row), po = __ldcg(q + 2 * ROWS + i);
                        const float v = fmaxf(mm, pm);
                        const float f0 = exp2_approx(mm - v), f1 = exp2_approx(pm - v);
                        acc = acc * f0 + po * f1;
                        ll = ll * f0 + pl * f1;
                        mm = v;
                    }
                    const int rr = rt * ROWS + row;
                    a.out[(long long)(r.row0 + rr / G) * a.out_stride + (long long)(h * G + rr % G) * D + d] =
                        bf16_bits(finish(acc, ll, a.cache.v_div));
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
constexpr int DECODE_ROWS = 16;

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
    w.prefill_parts = up(w.decode_parts + (long long)w.decode_blocks * 2 * DECODE_ROWS * (head_dim + 2) * 4);
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
