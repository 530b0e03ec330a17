// The 4-bit key/value cache: the step's plan (page tables, slot maps), the pass that norms and
// rotates the heads of q and k and writes k and v into the cache, and the exact read of rows.
// Formats and layout: kv4.cuh.
#include "common.cuh"
#include "kv4.cuh"

namespace vx {

static int kv4_sms() {
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

// ---- the plan of a step ------------------------------------------------------------------------
//
// Two prefix sums over the requests (new tokens, new pages) and then independent writes. Every
// block repeats the sums (8 bytes per request from L2, a block scan per PLAN_T requests) and
// writes its share: the requests with index % grid == block, new pages in turn, and one slice of the token rows. A new
// page's id is read from the free list, never back from the table, so no block waits for another;
// only `taken` needs an order when it is updated in place: the last block to have read it writes it.
constexpr int PLAN_T = 512;

__device__ __forceinline__ long long plan_scan(long long v, long long* warp_sums, long long& total) {
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if ((threadIdx.x & 31) >= o) x += y;
    }
    if ((threadIdx.x & 31) == 31) warp_sums[threadIdx.x >> 5] = x;
    __syncthreads();
    long long before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < PLAN_T / 32; i++) {
        const long long s = warp_sums[i];
        before += i < (int)(threadIdx.x >> 5) ? s : 0;
        total += s;
    }
    __syncthreads();
    return before + x - v;   // exclusive
}

__global__ void __launch_bounds__(PLAN_T)
kv4_plan_kernel(const int32_t* __restrict__ cached, const int32_t* __restrict__ fresh, int requests, int32_t* table,
                int cols, const int32_t* __restrict__ free_pages, int n_free, const int32_t* taken, int32_t* taken_out,
                int page_size, int tokens, int32_t* __restrict__ cu, int32_t* __restrict__ kv_lens,
                int32_t* __restrict__ positions, int32_t* __restrict__ slots, int32_t* __restrict__ status,
                uint32_t* ticket) {
    __shared__ long long warp_sums[PLAN_T / 32];
    __shared__ long long s_cu[PLAN_T + 1], s_at[PLAN_T];
    __shared__ int s_c[PLAN_T];
    __shared__ int s_flags;
    if (threadIdx.x == 0) {
        s_flags = 0;
        grid_launch_dependents();
    }
    grid_dependency_wait();
    const long long used = max(0, *taken);
    const long long slice = ((long long)tokens + gridDim.x - 1) / gridDim.x;
    const long long t_begin = blockIdx.x * slice, t_end = min((long long)tokens, t_begin + slice);
    const int P = page_size;
    long long tok0 = 0, need0 = 0;   // sums over the chunks before this one
    for (int base = 0; base < requests; base += PLAN_T) {
        const int b = base + threadIdx.x;
        long long c = 0, n = 0;
        if (b < requests) {
            c = max(0, cached[b]);
            n = max(0, fresh[b]);
        }
        const long long have = (c + P - 1) / P, full = (c + n + P - 1) / P;
        const long long want = min(full, (long long)cols), need = max(want - have, 0LL);
        long long tok_sum, need_sum;
        const long long tok = tok0 + plan_scan(n, warp_sums, tok_sum);
        const long long at = used + need0 + plan_scan(need, warp_sums, need_sum);
        s_cu[threadIdx.x] = tok;
        if (threadIdx.x == 0) s_cu[PLAN_T] = tok0 + tok_sum;
        s_at[threadIdx.x] = at;
        s_c[threadIdx.x] = (int)c;
        if (b < requests && full > cols) s_flags = 2;
        if (b < requests && b % gridDim.x == blockIdx.x) {
            cu[b] = (int32_t)tok;
            kv_lens[b] = (int32_t)min(c + n, (have + min(need, max(0LL, n_free - at))) * P);
        }
        __syncthreads();
        const int here = min(PLAN_T, requests - base);
        // this chunk's new pages, spread over all blocks
        for (long long i = (long long)blockIdx.x * PLAN_T + threadIdx.x; i < need_sum; i += (long long)gridDim.x * PLAN_T) {
            const long long at_i = used + need0 + i;
            int l = 0, r = here;   // last request whose first new page is <= at_i (those that need none share its start)
            while (r - l > 1) {
                const int m = (l + r) >> 1;
                if (s_at[m] <= at_i) l = m; else r = m;
            }
            const long long h = ((long long)s_c[l] + P - 1) / P;
            table[(long long)(base + l) * cols + h + (at_i - s_at[l])] = at_i < n_free ? free_pages[at_i] : -1;
        }
        // this chunk's token rows that fall into this block's slice
        const long long lo = max(t_begin, tok0), hi = min(t_end, tok0 + tok_sum);
        for (long long t = lo + threadIdx.x; t < hi; t += PLAN_T) {
            int l = 0, r = here;   // last request whose first row is <= t
            while (r - l > 1) {
                const int m = (l + r) >> 1;
                if (s_cu[m] <= t) l = m; else r = m;
            }
            const long long cc = s_c[l], p = cc + t - s_cu[l];
            const long long pi = p / P, h = (cc + P - 1) / P;
            int id = -1;
            if (pi < cols) {
                if (pi < h) {
                    id = table[(long long)(base + l) * cols + pi];
                } else {
                    const long long src = s_at[l] + pi - h;
                    id = src < n_free ? free_pages[src] : -1;
                }
            }
            positions[t] = (int32_t)p;
            slots[t] = id < 0 ? -1 : (int32_t)((long long)id * P + p % P);
        }
        tok0 += tok_sum;
        need0 += need_sum;
        __syncthreads();
    }
    for (long long t = max(t_begin, tok0) + threadIdx.x; t < t_end; t += PLAN_T) {
        positions[t] = -1;
        slots[t] = -1;
    }
    if (threadIdx.x == 0) {
        if (blockIdx.x == 0) {
            cu[requests] = (int32_t)tok0;
            *status = (used + need0 > n_free ? 1 : 0) | s_flags | (tok0 > tokens ? 4 : 0);
        }
        __threadfence();
        const uint32_t seen = atomicAdd(ticket, 1u);
        if (seen == gridDim.x - 1) {   // every block has read `taken`
            *ticket = 0;
            *taken_out = (int32_t)min(used + need0, (long long)n_free);
        }
    }
}

int kv4_plan(const int32_t* cached, const int32_t* fresh, int requests, int32_t* table, int cols,
             const int32_t* free_pages, int n_free, const int32_t* taken, int32_t* taken_out, int page_size, int tokens,
             int32_t* cu, int32_t* kv_lens, int32_t* positions, int32_t* slots, int32_t* status, uint32_t* ticket) {
    // about two token rows per thread, and no block without requests or rows
    int blocks = (tokens + 2 * PLAN_T - 1) / (2 * PLAN_T);
    const int by_requests = (requests + 127) / 128;
    if (blocks < by_requests) blocks = by_requests;
    if (blocks > 64) blocks = 64;
    if (blocks < 1) blocks = 1;
    EarlyLaunch l(blocks, PLAN_T);
    cudaLaunchKernelEx(&l.cfg, kv4_plan_kernel, cached, fresh, requests, table, cols, free_pages, n_free, taken, taken_out,
                       page_size, tokens, cu, kv_lens, positions, slots, status, ticket);
    return launch_status();
}

// ---- norms, rotation, quantised store ------------------------------------------------------------
//
// A row (one head of one token) is held by D/8 lanes, eight consecutive values each; a warp takes
// 32 / (D/8) rows at once and ROWS of those row groups of one token, so the token's cosines and
// sines are loaded once for all of them and every row's loads are in flight together.
//   q: x / sqrt(mean(x^2) + eps) * (offset + w), rotated; f32 throughout, rounded once.
//   k on its way into the cache: the same in f64. A 4-bit code changes by a whole step when the value
//   before it crosses a border, so the value handed to the quantiser is the correctly rounded f32 of
//   the formula: the cache's bytes then do not depend on how a sum was ordered.
//   The quantiser is the library's (actquant.cu): s = e4m3(divisor * amax / 6), code =
//   e2m1(x * divisor / s), single-precision steps.

template <typename T>
__device__ __forceinline__ T rope_sqrt_inv(T mean_eps);
template <>
__device__ __forceinline__ float rope_sqrt_inv<float>(float v) { return __fdiv_rn(1.0f, __fsqrt_rn(v)); }
template <>
__device__ __forceinline__ double rope_sqrt_inv<double>(double v) { return 1.0 / sqrt(v); }

// Norm and rotation of a row's eight values in this lane, in T.
template <typename T, int LPR>
__device__ __forceinline__ void norm_rotate(T (&x)[8], const float* __restrict__ weight, int offset, float eps,
                                            const float (&cs)[16], int rot, int interleaved, int li, bool rotate) {
    constexpr int D = LPR * 8;
    if (weight) {
        T ss = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) ss += x[i] * x[i];
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const T inv = rope_sqrt_inv<T>(ss / (T)D + (T)eps);
        const float4 w0 = *reinterpret_cast<const float4*>(weight + li * 8);
        const float4 w1 = *reinterpret_cast<const float4*>(weight + li * 8 + 4);
        const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = x[i] * inv * (offset ? (T)1 + (T)w[i] : (T)w[i]);
    }
    if (!rotate) return;   // uniform over the warp
    const bool mine = li * 8 < rot;
    if (interleaved) {
        if (mine) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const T c = (T)cs[i], s = (T)cs[8 + i], a = x[2 * i], b = x[2 * i + 1];
                x[2 * i] = a * c - b * s;
                x[2 * i + 1] = b * c + a * s;
            }
        }
    } else {
        const int half_lanes = rot / 16;
        const bool first = li < half_lanes;
        const int partner = (threadIdx.x & 31) + (mine ? (first ? half_lanes : -half_lanes) : 0);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const T o = __shfl_sync(0xffffffffu, x[i], partner);
            const T c = (T)cs[i], s = (T)cs[8 + i];
            if (mine) x[i] = first ? x[i] * c - o * s : x[i] * c + o * s;
        }
    }
}

__device__ __forceinline__ void load_row8(const void* p, long long at, int f32, float (&x)[8]) {
    if (f32) {
        const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at);
        const float4 b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + at);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ void store_row8(void* p, long long at, int f32, const float (&x)[8]) {
    if (f32) {
        float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + at);
        o[0] = make_float4(x[0], x[1], x[2], x[3]);
        o[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 v = __float22bfloat162_rn(make_float2(x[2 * i], x[2 * i + 1]));
            u[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + at) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// Quantises this lane's eight values (two neighbouring lanes make a group of 16).
__device__ __forceinline__ uint32_t quant8(const float (&x)[8], float divisor, uint32_t& scale) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    scale = f32_to_e4m3(__fdiv_rn(__fmul_rn(divisor, amax), 6.0f));
    uint32_t codes = 0;
    if (scale != 0) {
        const float ds = e4m3_to_f32(scale);
#pragma unroll
        for (int i = 0; i < 4; i++)
            codes |= f32x2_to_e2m1x2(__fdiv_rn(__fmul_rn(x[2 * i], divisor), ds),
                                     __fdiv_rn(__fmul_rn(x[2 * i + 1], divisor), ds)) << (8 * i);
    }
    return codes;
}

constexpr int ROPE_T = 128;

template <int LPR, int ROWS>
__global__ void __launch_bounds__(ROPE_T)
kv4_norm_rope_kernel(Kv4RopeArgs a) {
    constexpr int D = LPR * 8, RPG = 32 / LPR;   // rows per group
    const int lane = threadIdx.x & 31, li = lane % LPR, sub = lane / LPR;
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    const int gq = (a.heads + RPG - 1) / RPG, gk = (a.kv_heads + RPG - 1) / RPG;
    const int groups = gq + gk + (a.store ? gk : 0);
    const int chunks = (groups + ROWS - 1) / ROWS;
    const long long task = (long long)blockIdx.x * (ROPE_T / 32) + (threadIdx.x >> 5);
    if (task >= (long long)a.tokens * chunks) return;
    const long long tok = task / chunks;
    const int g0 = (int)(task - tok * chunks) * ROWS;
    const int pos = a.positions ? a.positions[tok] : 0;
    const int slot = a.store ? a.slots[tok] : 0;
    const long long slots = a.store ? a.cache.pages * a.cache.page_size : 0;
    // a row behind the last sequence, or outside the table: left as it was
    const bool live = pos >= 0 && (a.rope == nullptr || pos < a.rope_len);
    if (!live) return;
    const bool keep = a.store && slot >= 0 && slot < slots;

    float x[ROWS][8];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int g = g0 + r;
        const int kind = g < gq ? 0 : (g < gq + gk ? 1 : 2);
        const int head = (g - (kind == 0 ? 0 : kind == 1 ? gq : gq + gk)) * RPG + sub;
        const bool on = g < groups && head < (kind == 0 ? a.heads : a.kv_heads);
        if (on) {
            const void* p = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
            const long long st = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
            load_row8(p, tok * st + head * D + li * 8, a.in_f32, x[r]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[r][i] = 0.0f;
        }
    }
    float cs[16] = {};
    if (a.rope && li * 8 < a.rot) {
        const float* row = a.rope + (long long)pos * a.rot;
        if (a.interleaved) {   // four pairs
            const float4 c = *reinterpret_cast<const float4*>(row + li * 4);
            const float4 s = *reinterpret_cast<const float4*>(row + a.rot / 2 + li * 4);
            cs[0] = c.x; cs[1] = c.y; cs[2] = c.z; cs[3] = c.w;
            cs[8] = s.x; cs[9] = s.y; cs[10] = s.z; cs[11] = s.w;
        } else {
            const int at = li * 8 % (a.rot / 2);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float4 c = *reinterpret_cast<const float4*>(row + at + 4 * i);
                const float4 s = *reinterpret_cast<const float4*>(row + a.rot / 2 + at + 4 * i);
                cs[4 * i] = c.x; cs[4 * i + 1] = c.y; cs[4 * i + 2] = c.z; cs[4 * i + 3] = c.w;
                cs[8 + 4 * i] = s.x; cs[9 + 4 * i] = s.y; cs[10 + 4 * i] = s.z; cs[11 + 4 * i] = s.w;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int g = g0 + r;   // uniform over the warp
        if (g >= groups) break;
        const int kind = g < gq ? 0 : (g < gq + gk ? 1 : 2);
        const int head = (g - (kind == 0 ? 0 : kind == 1 ? gq : gq + gk)) * RPG + sub;
        const bool on = head < (kind == 0 ? a.heads : a.kv_heads);
        if (kind == 0 || (kind == 1 && !a.store)) {
            norm_rotate<float, LPR>(x[r], kind == 0 ? a.q_weight : a.k_weight, a.offset, a.eps, cs, a.rot, a.interleaved, li,
                                    a.rope != nullptr);
            if (on) store_row8(kind == 0 ? a.q_out : a.k_out, tok * (kind == 0 ? a.q_out_stride : a.k_out_stride) + head * D + li * 8,
                               a.out_f32, x[r]);
            continue;
        }
        if (kind == 1 && (a.k_weight || a.rope)) {
            double y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = (double)x[r][i];
            norm_rotate<double, LPR>(y, a.k_weight, a.offset, a.eps, cs, a.rot, a.interleaved, li, a.rope != nullptr);
#pragma unroll
            for (int i = 0; i < 8; i++) x[r][i] = (float)y[i];
        }
        uint32_t scale;
        const uint32_t codes = quant8(x[r], kind == 1 ? a.cache.k_div : a.cache.v_div, scale);
        if (on && keep) {
            int tau;
            uint8_t* blk = kv4_block_of(a.cache, slot, head, tau);
            // (eight values = four code bytes; a V piece of D/16 bytes holds two or one such words)
            *reinterpret_cast<uint32_t*>(blk + (kind == 1 ? kv4_k_code(D, tau, li * 4) : kv4_v_code(D, tau, li * 4))) = codes;
            if ((li & 1) == 0) blk[kind == 1 ? kv4_k_scale(D, tau, li >> 1) : kv4_v_scale(D, tau, li >> 1)] = (uint8_t)scale;
        }
    }
}

int kv4_norm_rope(const Kv4RopeArgs& a) {
    const int rpg = 256 / a.head_dim;
    const int gq = (a.heads + rpg - 1) / rpg, gk = (a.kv_heads + rpg - 1) / rpg;
    const int groups = gq + gk * (a.store ? 2 : 1);
    // Several row groups per warp once there are enough warps to fill the machine without it (four
    // blocks of four warps per SM).
    const int rows = (long long)a.tokens * ((groups + 3) / 4) >= 16LL * kv4_sms() ? 4 : 1;
    const long long warps = (long long)a.tokens * ((groups + rows - 1) / rows);
    const long long blocks = (warps + ROPE_T / 32 - 1) / (ROPE_T / 32);
    if (blocks > 0x7fffffffLL) return VELOX_ERR_UNSUPPORTED;
    EarlyLaunch l((unsigned)blocks, ROPE_T);
#define VX_ROPE(LPR)                                                          \
    if (rows == 4) cudaLaunchKernelEx(&l.cfg, kv4_norm_rope_kernel<LPR, 4>, a); \
    else cudaLaunchKernelEx(&l.cfg, kv4_norm_rope_kernel<LPR, 1>, a);
    if (a.head_dim == 128) {
        VX_ROPE(16)
    } else {
        VX_ROPE(8)
    }
#undef VX_ROPE
    return launch_status();
}

// ---- exact read of rows ---------------------------------------------------------------------------
// One thread per eight values of a row (four code bytes): value = (code * scale) / divisor; the
// product is exact (six significant bits), the quotient is rounded once to f32, then to the output.
__global__ void __launch_bounds__(256)
kv4_rows_kernel(Kv4Geom c, const int32_t* __restrict__ slots, int tokens, void* k_out, void* v_out, int out_f32) {
    const int D = c.head_dim, per_row = D / 8;
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    const long long rows = (long long)tokens * c.kv_heads;
    const long long total = rows * per_row * 2, cap = c.pages * c.page_size;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const bool is_v = i >= total / 2;
        const long long e = is_v ? i - total / 2 : i;
        void* dst = is_v ? v_out : k_out;
        if (!dst) continue;
        const long long row = e / per_row;
        const int w = (int)(e - row * per_row);
        const long long tok = row / c.kv_heads;
        const int h = (int)(row - tok * c.kv_heads);
        const int slot = slots[tok];
        if (slot < 0 || slot >= cap) continue;   // a row that is not in the cache: left as it was
        int tau;
        const uint8_t* blk = kv4_block_of(c, slot, h, tau);
        const uint32_t codes = *reinterpret_cast<const uint32_t*>(blk + (is_v ? kv4_v_code(D, tau, w * 4) : kv4_k_code(D, tau, w * 4)));
        const float s = e4m3_to_f32(blk[is_v ? kv4_v_scale(D, tau, w >> 1) : kv4_k_scale(D, tau, w >> 1)] & 0x7fu);
        const float div = is_v ? c.v_div : c.k_div;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = __fdiv_rn(e2m1_to_f32(codes >> (4 * j) & 15u) * s, div);
        store_row8(dst, row * D + w * 8, out_f32, x);
    }
}

int kv4_rows(const Kv4Geom& c, const int32_t* slots, int tokens, void* k_out, void* v_out, int out_f32) {
    const long long total = (long long)tokens * c.kv_heads * (c.head_dim / 8) * 2;
    long long blocks = (total + 255) / 256;
    if (blocks > 16LL * kv4_sms()) blocks = 16LL * kv4_sms();
    EarlyLaunch l((unsigned)blocks, 256);
    cudaLaunchKernelEx(&l.cfg, kv4_rows_kernel, c, slots, tokens, k_out, v_out, out_f32);
    return launch_status();
}

}  // namespace vx
