// The 4-bit key/value cache: geometry of its blocks and the argument structs of its kernels.
//
// Values are NVFP4 as in the weights and activations of this library (E2M1 codes, one E4M3 scale per
// 16 values, a divisor per tensor: value = code * scale / divisor), 4.5 bits each. A page holds
// page_size tokens; per page and kv head it is a run of page_size / 16 blocks. A block is 16 tokens
// of K and V, 18 * D bytes, laid out so that lane (g, t) = (lane / 4, lane % 4) of a warp reads its
// operands of the m16n8k16 MMA with one access per plane at lane * (access size), straight from
// global memory:
//   [0, 8D)     K codes: token-major, D/2 bytes per token. Lane (g, t): tokens g and g + 8, dimensions
//               t*D/4 .. (t+1)*D/4 (the order along the contraction does not matter).
//   [8D, 16D)   V codes: D/16-byte pieces [p][g][t][j] = token 8p + 2t + j, dimensions g*D/8 ..: the
//               four tokens whose probabilities the MMA hands to lane (g, t).
//   [16D, 17D)  K scales [r][t][h][i]: token 8h + r, group t*D/64 + i.
//   [17D, 18D)  V scales [group][t][p][j].
// Every byte pattern decodes to a finite number (a scale byte is read as seven magnitude bits, 0x7f
// as 480), so bytes that no token has written cannot put a NaN into a product with a zero
// probability.
#pragma once

#include "common.cuh"

namespace vx {

struct Kv4Geom {
    uint8_t* blocks;
    long long pages;
    int page_size, page_shift, kv_heads, head_dim;   // page_size = 1 << page_shift
    float k_div, v_div;
};

__host__ __device__ __forceinline__ int kv4_block_bytes(int head_dim) { return 18 * head_dim; }

// Start of the block that holds `slot` (= page * page_size + offset) of head h, and the token's
// place in it.
__device__ __forceinline__ uint8_t* kv4_block_of(const Kv4Geom& c, int slot, int h, int& tau) {
    const int off = slot & (c.page_size - 1);
    tau = off & 15;
    const long long chunk = (long long)(slot >> c.page_shift) * c.kv_heads + h;
    return c.blocks + ((chunk << (c.page_shift - 4)) + (off >> 4)) * kv4_block_bytes(c.head_dim);
}
// Offsets of a token's pieces inside its block. `byte` counts the code bytes of a row (D/2 of them).
__device__ __forceinline__ int kv4_k_code(int D, int tau, int byte) { return tau * (D / 2) + byte; }
__device__ __forceinline__ int kv4_v_code(int D, int tau, int byte) {
    const int piece = D / 16, g = byte / piece;
    return 8 * D + (((((tau >> 3) * 8 + g) * 4 + ((tau >> 1) & 3)) * 2 + (tau & 1)) * piece) + byte % piece;
}
__device__ __forceinline__ int kv4_k_scale(int D, int tau, int group) {
    const int per = D / 64;
    return 16 * D + (((tau & 7) * 4 + group / per) * 2 + (tau >> 3)) * per + group % per;
}
__device__ __forceinline__ int kv4_v_scale(int D, int tau, int group) {
    return 17 * D + ((group * 4 + ((tau >> 1) & 3)) * 2 + (tau >> 3)) * 2 + (tau & 1);
}

struct Kv4RopeArgs {
    const void *q, *k, *v;        // [tokens, heads, D], row strides below; f32 or bf16 (in_f32)
    long long q_stride, k_stride, v_stride;
    int in_f32;
    const float *q_weight, *k_weight;   // NULL: no norm
    const float* rope;                  // [positions, rot]: cosines, then sines; NULL: no rotation
    int rope_len, rot, interleaved;
    const int32_t* positions;
    const int32_t* slots;               // cache form only
    void *q_out, *k_out;                // NULL k_out in the cache form
    long long q_out_stride, k_out_stride;
    int out_f32;
    int tokens, heads, kv_heads, head_dim;
    float eps;
    int offset;
    int store;                          // write k and v into the cache
    Kv4Geom cache;
};
int kv4_norm_rope(const Kv4RopeArgs& a);

int kv4_plan(const int32_t* cached, const int32_t* fresh, int requests, int32_t* table, int cols,
             const int32_t* free_pages, int n_free, const int32_t* taken, int32_t* taken_out, int page_size, int tokens,
             int32_t* cu, int32_t* kv_lens, int32_t* positions, int32_t* slots, int32_t* status, uint32_t* ticket);

int kv4_rows(const Kv4Geom& c, const int32_t* slots, int tokens, void* k_out, void* v_out, int out_f32);

struct Kv4AttnArgs {
    const uint16_t* q;                  // [tokens, heads, D] bf16
    long long q_stride;
    uint16_t* out;
    long long out_stride;
    Kv4Geom cache;
    const int32_t* table;               // [requests, cols]
    int cols;
    const int32_t* cu;                  // [requests + 1]
    const int32_t* kv_lens;             // [requests]
    int requests, tokens, heads;
    float scale;
    int causal, window;
    int max_new;
    uint8_t* ws;
    // set by the dispatcher: requests a kernel takes, by query rows per kv head: (min_rows, max_rows]; and where the
    // parts of the decode kernel's split items lie in the workspace (its tickets are at the start)
    int min_rows, max_rows;
    long long decode_parts, prefill_tickets, prefill_parts;
};
long long kv4_attention_workspace(int head_dim);
int kv4_attention(Kv4AttnArgs a);
// many query rows per request, on the tcgen05 tensor cores
int kv4_prefill(const Kv4AttnArgs& a, int blocks);
long long kv4_prefill_parts_bytes(int blocks, int head_dim);
int kv4_status_sync();
int kv4_status_reset();

}  // namespace vx
