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
// Bound by latency: 5 us for 64 requests, 10 us for 1000 with 35,000 rows (dependent loads, two block scans per
// 512 requests).
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
    const int P = page_size, sh = __ffs(page_size) - 1;   // (a power of two; 64-bit divisions are slow)
    long long tok0 = 0, need0 = 0;   // sums over the chunks before this one
    for (int base = 0; base < requests; base += PLAN_T) {
        const int b = base + threadIdx.x;
        long long c = 0, n = 0;
        if (b < requests) {
            c = max(0, cached[b]);
            n = max(0, fresh[b]);
        }
        const long long have = (c + P - 1) >> sh, full = (c + n + P - 1) >> sh;
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
            kv_lens[b] = (int32_t)min(0x7fffffffLL, min(c + n, (have + min(need, max(0LL, n_free - at))) * P));
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
            const long long h = ((long long)s_c[l] + P - 1) >> sh;
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
            const long long pi = p >> sh, h = (cc + P - 1) >> sh;
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
            const long long slot = (long long)id * P + (p & (P - 1));
            slots[t] = id < 0 || slot > 0x7fffffffLL ? -1 : (int32_t)slot;
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
// 32 / (D/8) rows at once. A task is ROWS such groups of q rows of one token, or as many of its k and v rows, so
// the token's cosines and sines are loaded once per task. Warps walk the tasks with the grid's stride, all q tasks
// first, and request the next task's rows before they finish this one's. With one task per warp the pass waited
// for three memory round trips per 2 KB (2048 tokens of 64 + 8 + 8 heads, bf16: 73 us); with q, k and v rows mixed
// in a task the warps that met the k rows (f64) every time ended last (75 us). Now 26 us, bound by instructions (more
// than an issue slot in two is used; its 77 MB are 12 us).
//   q: x / sqrt(mean(x^2) + eps) * (offset + w), rotated; f32 throughout, rounded once.
//   k on its way into the cache: the same in f64. A 4-bit code changes by a whole step when the value
//   before it crosses a border, so the value handed to the quantiser is the correctly rounded f32 of
//   the formula: the cache's bytes then do not depend on how a sum was ordered.
//   The quantiser is the library's (actquant.cu): s = e4m3(divisor * amax / 6), code =
//   e2m1(x * divisor / s), single-precision steps.

__device__ __forceinline__ void unpack8(const uint4& a, float (&x)[8]) {
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack8(const uint4& a, const uint4& b, float (&x)[8]) {
    const uint32_t u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __uint_as_float(u[i]);
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

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// What a lane needs of the rotation of its eight dimensions: y = c x + s (its partner's x), with the sign in s. Pairs
// of neighbours are in the lane itself (the first four entries); a lane that is not rotated has c = 1, s = 0 and
// itself as the partner.
struct Turn {
    float c[8], s[8];
    int partner;
};

template <typename T>
__device__ __forceinline__ void rotate8(T (&x)[8], const Turn& t, int interleaved) {
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const T a = x[2 * i], b = x[2 * i + 1], c = (T)t.c[i], s = (T)t.s[i];
            x[2 * i] = a * c - b * s;
            x[2 * i + 1] = b * c + a * s;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const T o = __shfl_sync(0xffffffffu, x[i], t.partner);
            x[i] = x[i] * (T)t.c[i] + o * (T)t.s[i];
        }
    }
}

template <int LPR>
__device__ __forceinline__ void norm8_f32(float (&x)[8], const float* __restrict__ weight, int offset, float eps, int li) {
    constexpr int D = LPR * 8;
    float w[8];
    load8(weight + li * 8, w);
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float inv = rsqrtf(ss * (1.0f / D) + eps);   // (two units in the last place at most)
    if (offset) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] += 1.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = x[i] * inv * w[i];
}

// The same in f64. 1 / sqrt by two Newton steps from the single-precision estimate (2^-22 -> 2^-44 -> 2^-88): a
// few units of 2^-53.
template <int LPR>
__device__ __forceinline__ void norm8_f64(double (&x)[8], const float* __restrict__ weight, int offset, float eps, int li) {
    constexpr int D = LPR * 8;
    float w[8];
    load8(weight + li * 8, w);
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) ss = fma(x[i], x[i], ss);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const double v = ss * (1.0 / D) + (double)eps;
    double inv;
    // (estimates outside f32's range, for sums that a norm never sees in earnest, take the plain route)
    if (v > 1e-30 && v < 1e30) {
        inv = (double)rsqrtf((float)v);
#pragma unroll
        for (int i = 0; i < 2; i++) inv = inv * fma(-0.5 * v * inv, inv, 1.5);
    } else {
        inv = 1.0 / sqrt(v);
    }
    const double one = offset ? 1.0 : 0.0;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = x[i] * inv * (one + (double)w[i]);
}

// a / b for normal quotients from r = 1 / b: one correction of the rounded product gives the correctly
// rounded quotient.
__device__ __forceinline__ float quotient(float a, float b, float r) {
    const float q = a * r;
    return fmaf(fmaf(-q, b, a), r, q);
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
        const float ds = e4m3_to_f32(scale), r = __fdiv_rn(1.0f, ds);
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; i++)   // (past 1e30 a value saturates at any scale; kept finite for the correction)
            q[i] = quotient(fminf(fmaxf(__fmul_rn(x[i], divisor), -1e30f), 1e30f), ds, r);
#pragma unroll
        for (int i = 0; i < 4; i++) codes |= f32x2_to_e2m1x2(q[2 * i], q[2 * i + 1]) << (8 * i);
    }
    return codes;
}

constexpr int ROPE_T = 128;
// Row groups per task once there is work for every warp, and blocks per SM that this leaves room for.
constexpr int rope_rows(bool f32) { return f32 ? 2 : 4; }
constexpr int rope_blocks(int rows) { return rows == 1 ? 8 : 5; }

template <int LPR, int ROWS, bool F32>
__global__ void __launch_bounds__(ROPE_T, rope_blocks(ROWS))
kv4_norm_rope_kernel(const __grid_constant__ Kv4RopeArgs a) {
    constexpr int D = LPR * 8, RPG = 32 / LPR;   // rows per group
    const int lane = threadIdx.x & 31, li = lane % LPR, sub = lane / LPR;
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    // Tasks of a token: cq of q rows, then ck of k rows, or of k and v rows in turn where they are stored.
    const unsigned gq = (a.heads + RPG - 1) / RPG, gk = (a.kv_heads + RPG - 1) / RPG * (a.store ? 2 : 1);
    const unsigned cq = (gq + ROWS - 1) / ROWS, ck = (gk + ROWS - 1) / ROWS;
    const unsigned tq = (unsigned)a.tokens * cq, total = tq + (unsigned)a.tokens * ck, stride = gridDim.x * (ROPE_T / 32);
    const long long slots = a.store ? a.cache.pages * a.cache.page_size : 0;

    struct Task {
        uint4 x[ROWS][F32 ? 2 : 1];
        int pos, slot;
        unsigned tok, g0;
    };
    // Group g of a token's k / v rows: the k and the v row of a head group follow each other. A lane's place in a group
    // of rows is lane * 8 elements in, the next group of the same operand 256 elements on.
    auto head_of = [&](bool q, unsigned g) { return (int)(q || !a.store ? g : g >> 1) * RPG + sub; };
    auto fetch = [&](unsigned task, Task& t) {
        const bool q = task < tq;
        if (!q) task -= tq;
        t.tok = task / (q ? cq : ck);
        t.g0 = (task - t.tok * (q ? cq : ck)) * ROWS;
        t.pos = a.positions ? a.positions[t.tok] : 0;
        t.slot = a.store ? a.slots[t.tok] : 0;
        const int bytes = F32 ? 4 : 2, heads = q ? a.heads : a.kv_heads;
        const bool both = !q && a.store;
        const uint8_t* at = reinterpret_cast<const uint8_t*>(q ? a.q : a.k) +
                            ((long long)t.tok * (q ? a.q_stride : a.k_stride) + (both ? t.g0 >> 1 : t.g0) * 256 + lane * 8) * bytes;
        const uint8_t* at_v = at;
        if (both) at_v = reinterpret_cast<const uint8_t*>(a.v) + ((long long)t.tok * a.v_stride + (t.g0 >> 1) * 256 + lane * 8) * bytes;
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            const uint8_t* src = !both ? at + r * 256 * bytes : ((ROWS == 1 ? t.g0 : r) & 1 ? at_v : at) + (r >> 1) * 256 * bytes;
            const bool on = head_of(q, t.g0 + r) < heads;
#pragma unroll
            for (int i = 0; i < (F32 ? 2 : 1); i++)
                t.x[r][i] = on ? reinterpret_cast<const uint4*>(src)[i] : make_uint4(0, 0, 0, 0);
        }
    };

    unsigned task = blockIdx.x * (ROPE_T / 32) + (threadIdx.x >> 5);
    if (task >= total) return;
    Task next;
    fetch(task, next);
    for (bool more = true; more; task += stride) {
        const Task t = next;
        more = total - task > stride;
        // a row behind the last sequence, or outside the table: left as it was
        const bool live = t.pos >= 0 && (a.rope == nullptr || t.pos < a.rope_len);
        Turn turn;
        turn.partner = lane;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            turn.c[i] = 1.0f;
            turn.s[i] = 0.0f;
        }
        if (a.rope && live && li * 8 < a.rot) {
            const int half = a.rot / 2, half_lanes = a.rot / 16;
            const float* row = a.rope + (long long)t.pos * a.rot;
            if (a.interleaved) {   // four pairs
                const float4 c = *reinterpret_cast<const float4*>(row + li * 4), s = *reinterpret_cast<const float4*>(row + half + li * 4);
                turn.c[0] = c.x; turn.c[1] = c.y; turn.c[2] = c.z; turn.c[3] = c.w;
                turn.s[0] = s.x; turn.s[1] = s.y; turn.s[2] = s.z; turn.s[3] = s.w;
            } else {
                const bool first = li < half_lanes;
                turn.partner = lane + (first ? half_lanes : -half_lanes);
                load8(row + (first ? li : li - half_lanes) * 8, turn.c);
                load8(row + half + (first ? li : li - half_lanes) * 8, turn.s);
#pragma unroll
                for (int i = 0; i < 8; i++) turn.s[i] = first ? -turn.s[i] : turn.s[i];
            }
        }
        if (more) fetch(task + stride, next);
        if (!live) continue;   // uniform over the warp
        const bool q = task < tq;
        if (q || !a.store) {
            const float* weight = q ? a.q_weight : a.k_weight;
            const int heads = q ? a.heads : a.kv_heads;
            const long long at = (long long)t.tok * (q ? a.q_out_stride : a.k_out_stride) + t.g0 * 256 + lane * 8;
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const int head = (int)(t.g0 + r) * RPG + sub;
                float x[8];
                if (F32) unpack8(t.x[r][0], t.x[r][F32 ? 1 : 0], x); else unpack8(t.x[r][0], x);
                if (weight) norm8_f32<LPR>(x, weight, a.offset, a.eps, li);
                if (a.rope) rotate8(x, turn, a.interleaved);
                if (head < heads) store_row8(q ? a.q_out : a.k_out, at + r * 256, a.out_f32, x);
            }
        } else {
            const bool keep = t.slot >= 0 && t.slot < slots;
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const unsigned g = t.g0 + r;   // uniform over the warp
                const int head = head_of(false, g);
                const bool v = g & 1;
                float x[8];
                if (F32) unpack8(t.x[r][0], t.x[r][F32 ? 1 : 0], x); else unpack8(t.x[r][0], x);
                if (!v && (a.k_weight || a.rope)) {
                    double y[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] = (double)x[i];
                    if (a.k_weight) norm8_f64<LPR>(y, a.k_weight, a.offset, a.eps, li);
                    if (a.rope) rotate8(y, turn, a.interleaved);
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = (float)y[i];
                }
                uint32_t scale;
                const uint32_t codes = quant8(x, v ? a.cache.v_div : a.cache.k_div, scale);
                if (head < a.kv_heads && keep) {
                    int tau;
                    uint8_t* blk = kv4_block_of(a.cache, t.slot, head, tau);
                    // (eight values = four code bytes; a V piece of D/16 bytes holds two or one such words)
                    *reinterpret_cast<uint32_t*>(blk + (v ? kv4_v_code(D, tau, li * 4) : kv4_k_code(D, tau, li * 4))) = codes;
                    if ((li & 1) == 0) blk[v ? kv4_v_scale(D, tau, li >> 1) : kv4_k_scale(D, tau, li >> 1)] = (uint8_t)scale;
                }
            }
        }
    }
}

int kv4_norm_rope(const Kv4RopeArgs& a) {
    const int rpg = 256 / a.head_dim;
    const long long gq = (a.heads + rpg - 1) / rpg, gk = (a.kv_heads + rpg - 1) / rpg * (a.store ? 2 : 1);
    // Several row groups per task once there are enough tasks to fill the machine without it (four blocks of four
    // warps per SM).
    const int many = rope_rows(a.in_f32);
    auto tasks = [&](int rows) { return (long long)a.tokens * ((gq + rows - 1) / rows + (gk + rows - 1) / rows); };
    const int rows = tasks(many) >= 16LL * kv4_sms() ? many : 1;
    if (tasks(rows) > 0x7fffffffLL) return VELOX_ERR_UNSUPPORTED;
    const long long fit = (long long)rope_blocks(rows) * kv4_sms();
    long long blocks = (tasks(rows) + ROPE_T / 32 - 1) / (ROPE_T / 32);
    if (blocks > fit) blocks = fit;
    EarlyLaunch l((unsigned)blocks, ROPE_T);
#define VX_ROPE(LPR, F32)                                                                           \
    if (rows != 1) cudaLaunchKernelEx(&l.cfg, kv4_norm_rope_kernel<LPR, rope_rows(F32), F32>, a);   \
    else cudaLaunchKernelEx(&l.cfg, kv4_norm_rope_kernel<LPR, 1, F32>, a);
    if (a.head_dim == 128) {
        if (a.in_f32) { VX_ROPE(16, true) } else { VX_ROPE(16, false) }
    } else {
        if (a.in_f32) { VX_ROPE(8, true) } else { VX_ROPE(8, false) }
    }
#undef VX_ROPE
    return launch_status();
}

// ---- exact read of rows ---------------------------------------------------------------------------
// A warp takes the K and the V rows of 16 * 8 / D heads of a token, a lane eight values of a row (four
// code bytes): value = (code * scale) / divisor; the product is exact (six significant bits), the quotient
// rounded once to f32, then to the output's type.
template <int LPR>
__global__ void __launch_bounds__(256)
kv4_rows_kernel(Kv4Geom c, const int32_t* __restrict__ slots, int tokens, void* k_out, void* v_out, int out_f32) {
    constexpr int D = LPR * 8, HEADS = 16 / LPR;   // heads per warp
    if (threadIdx.x == 0) grid_launch_dependents();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, w = lane % LPR, is_v = (lane / LPR) & 1, sub = lane / (2 * LPR);
    const unsigned chunks = (c.kv_heads + HEADS - 1) / HEADS;
    const unsigned total = (unsigned)tokens * chunks, stride = gridDim.x * 8;
    const long long cap = c.pages * c.page_size;
    void* dst = is_v ? v_out : k_out;
    const float div = is_v ? c.v_div : c.k_div, r = __fdiv_rn(1.0f, div);
    for (unsigned task = blockIdx.x * 8 + (threadIdx.x >> 5); task < total; task += stride) {
        const unsigned tok = task / chunks;
        const int h = (int)(task - tok * chunks) * HEADS + sub;
        const int slot = slots[tok];
        if (slot >= 0 && slot < cap && h < c.kv_heads && dst) {   // (a row that is not in the cache: left as it was)
            int tau;
            const uint8_t* blk = kv4_block_of(c, slot, h, tau);
            const uint32_t codes = *reinterpret_cast<const uint32_t*>(blk + (is_v ? kv4_v_code(D, tau, w * 4) : kv4_k_code(D, tau, w * 4)));
            const float s = e4m3_to_f32(blk[is_v ? kv4_v_scale(D, tau, w >> 1) : kv4_k_scale(D, tau, w >> 1)] & 0x7fu);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = quotient(e2m1_to_f32(codes >> (4 * j) & 15u) * s, div, r);
            store_row8(dst, ((long long)tok * c.kv_heads + h) * D + w * 8, out_f32, x);
        }
    }
}

int kv4_rows(const Kv4Geom& c, const int32_t* slots, int tokens, void* k_out, void* v_out, int out_f32) {
    const int heads = c.head_dim == 128 ? 1 : 2;
    const long long tasks = (long long)tokens * ((c.kv_heads + heads - 1) / heads);
    if (tasks > 0x7fffffffLL) return VELOX_ERR_UNSUPPORTED;
    long long blocks = (tasks + 7) / 8;
    if (blocks > 8LL * kv4_sms()) blocks = 8LL * kv4_sms();
    EarlyLaunch l((unsigned)blocks, 256);
    if (c.head_dim == 128)
        cudaLaunchKernelEx(&l.cfg, kv4_rows_kernel<16>, c, slots, tokens, k_out, v_out, out_f32);
    else
        cudaLaunchKernelEx(&l.cfg, kv4_rows_kernel<8>, c, slots, tokens, k_out, v_out, out_f32);
    return launch_status();
}

}  // namespace vx
