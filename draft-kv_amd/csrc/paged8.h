// The full cache in 8 bits (dkv_paged8_t): layout, and the loads that the append, the attention and the drafter
// mirror's sync share.
//
// What a cache holds. Rows of K and V, rounded to bf16. Once all block_size rows of a block are there the block is
// sealed: per (KV head, K or V) a = max |x| over the block's finite values, e the least integer with a <= 448 * 2^e
// (0 where a = 0, within -126 .. 119), codes e4m3(x * 2^-e) to nearest even, saturating; NaN and infinities become the NaN code. The
// product with a power of two is exact, so a code is one rounding of the bf16 value, whatever the device.
//
// Who reads what. A query at position p reads the blocks before its own in 8 bits, and its own block's rows up to p in
// bf16. What it sees is a function of rows 0 .. p alone: not of how many rows share a call, of how they were appended,
// or of rejected rows that were there in between (their block's codes are written again when it fills again). That is
// what keeps greedy speculative decoding over this cache equal to plain decoding over it. The bf16 rows live in a ring
// per (sequence, layer), the last tail_rows rows; an append of more rows than fit beside the open block also leaves
// all its rows in `hot`, which the attention that follows reads instead. Its last rows then take the places of the open
// block's in the ring: those go to `held`, tile by tile with their position as a tag, so that the same append can be made
// again (a forward that failed, a state that is run again). A tag says that held has the tile's newest rows; whoever
// puts the tile's rows elsewhere takes it back.
//
// Tiles. 16 tokens of one (KV head, K or V), channels padded with zeros to DP = 32, 64, 128, 192 or 256, in panels of
// PW = min(64, DP) channels. A panel holds PW / 4 values per lane, lane-major, in the order of the matrix
// instruction's A operand: lane 16 q + c has
//     K: token c, channels PW i + (PW/4) q + 0 .. PW/4 - 1
//     V: channels PW i + 16 t + c, tokens 4 q .. 4 q + 3   (t major)
// so every load of a wave is one contiguous run (1 KB of codes), K and V go from memory to the matrix cores without
// passing through LDS, and V needs no transposition. Codes and bf16 rows use the same order.
#pragma once

#include "dkv_common.h"

namespace dkv {

constexpr int P8_MAXD = 256;

__host__ __device__ inline int p8_dp(int d) { return d <= 32 ? 32 : (d + 63) / 64 * 64; }
__host__ __device__ inline int64_t p8_block_bytes(int heads, int d, int bs) {
    return (int64_t)heads * bs * p8_dp(d) * 2 + (2 * heads + 15) / 16 * 16;
}
__host__ __device__ inline int64_t p8_row_bytes(int heads, int d) { return (int64_t)heads * p8_dp(d) * 4; }

// whether an append of T rows keeps them all in the ring, beside the open block's
__host__ __device__ inline bool p8_in_ring(const dkv_paged8_t& c, int T) {
    return (c.block_size - 1 + T + 15) / 16 * 16 <= c.tail_rows;
}
__host__ __device__ inline int p8_hot_rows(const dkv_paged8_t& c, int T) {
    return p8_in_ring(c, T) ? 0 : (c.block_size - 1 + T + 15) / 16 * 16;
}

// The rows that a call brings to a sequence: none where they would lie outside its block table.
__device__ __forceinline__ int p8_new_rows(const dkv_paged8_t& c, int T, int s0, const int32_t* count, int s) {
    const int n = count ? min(count[s], T) : T;
    return n <= 0 || s0 < 0 || (int64_t)s0 + n > (int64_t)c.max_blocks * c.block_size ? 0 : n;
}

// offset of a value in its tile
__device__ __forceinline__ int p8_k_off(int dp, int token, int d) {
    const int pw = dp < 64 ? dp : 64, pb = pw / 4, x = d % pw;
    return d / pw * 16 * pw + (x / pb * 16 + token) * pb + x % pb;
}
__device__ __forceinline__ int p8_v_off(int dp, int token, int d) {
    const int pw = dp < 64 ? dp : 64, pb = pw / 4, x = d % pw;
    return d / pw * 16 * pw + (token / 4 * 16 + x % 16) * pb + x / 16 * 4 + token % 4;
}

// bf16 tile (K; V follows it, 16 DP values on) of 16 rows from position pos (a multiple of 16)
__device__ __forceinline__ uint16_t* p8_ring_tile(const dkv_paged8_t& c, int s, int layer, int h, int pos) {
    const int64_t tiles = c.tail_rows / 16;
    return static_cast<uint16_t*>(c.tail) +
           ((((int64_t)s * c.n_layers + layer) * c.n_kv_heads + h) * tiles + pos % c.tail_rows / 16) * 32 * p8_dp(c.head_dim);
}
// the same in the hot rows of the call whose first open block starts at position base
__device__ __forceinline__ uint16_t* p8_hot_tile(const dkv_paged8_t& c, int s, int h, int pos, int base) {
    const int64_t tiles = c.hot_rows / 16;
    return static_cast<uint16_t*>(c.hot) +
           (((int64_t)s * c.n_kv_heads + h) * tiles + (pos - base) / 16) * 32 * p8_dp(c.head_dim);
}

// A tile of the open block in held [batch][layer][head][block_size / 16], and behind it a tag for each (K or V, panel):
// every one belongs to the one wave of an append that has that panel.
__host__ __device__ inline int p8_panels(int dp) { return dp < 64 ? 1 : dp / 64; }
__host__ __device__ inline int p8_held_stride(int dp) { return 64 * dp + (8 * p8_panels(dp) + 15) / 16 * 16; }
__device__ __forceinline__ uint16_t* p8_held_tile(const dkv_paged8_t& c, int s, int layer, int h, int pos) {
    const int64_t tile = (((int64_t)s * c.n_layers + layer) * c.n_kv_heads + h) * (c.block_size / 16) + pos % c.block_size / 16;
    return reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(c.held) + tile * p8_held_stride(p8_dp(c.head_dim)));
}
__device__ __forceinline__ int32_t* p8_held_tag(const dkv_paged8_t& c, int s, int layer, int h, int pos, int kv, int panel) {
    const int dp = p8_dp(c.head_dim);
    return reinterpret_cast<int32_t*>(p8_held_tile(c, s, layer, h, pos) + 32 * dp) + kv * p8_panels(dp) + panel;
}
// bf16 tile at pos of the open block (outside an append all panels' tags agree)
__device__ __forceinline__ const uint16_t* p8_open_tile(const dkv_paged8_t& c, int s, int layer, int h, int pos) {
    return c.held && *p8_held_tag(c, s, layer, h, pos, 0, 0) == pos ? p8_held_tile(c, s, layer, h, pos)
                                                                     : p8_ring_tile(c, s, layer, h, pos);
}

__device__ __forceinline__ const uint8_t* p8_block(const dkv_paged8_t& c, int s, int layer, int pos) {
    return static_cast<const uint8_t*>(c.pool) +
           c.block_table[((int64_t)s * c.n_layers + layer) * c.max_blocks + pos / c.block_size] *
               p8_block_bytes(c.n_kv_heads, c.head_dim, c.block_size);
}
// byte offset in a block of the tile of 16 tokens from `off` of a head; V's follows 16 DP on
__device__ __forceinline__ int64_t p8_tile_off(const dkv_paged8_t& c, int h, int off) {
    return ((int64_t)h * (c.block_size / 16) + off / 16) * 32 * p8_dp(c.head_dim);
}
// offset of a head's two exponent bytes (K, V), biased by 127, behind the block's tiles
__device__ __forceinline__ int64_t p8_scale_off(const dkv_paged8_t& c, int h) {
    return (int64_t)c.n_kv_heads * c.block_size * p8_dp(c.head_dim) * 2 + 2 * h;
}

__device__ __forceinline__ float p8_scale(uint32_t biased) { return __uint_as_float(biased << 23); }

// one value of a sequence that holds `len` rows (kv: 0 K, 1 V); pos < len
__device__ __forceinline__ float p8_value(const dkv_paged8_t& c, int s, int layer, int pos, int len, int h, int d, int kv) {
    const int dp = p8_dp(c.head_dim);
    const int o = (kv ? p8_v_off(dp, pos % 16, d) : p8_k_off(dp, pos % 16, d)) + kv * 16 * dp;
    if (pos >= len / c.block_size * c.block_size) return bf16_to_f32(p8_open_tile(c, s, layer, h, pos / 16 * 16)[o]);
    const uint8_t* b = p8_block(c, s, layer, pos);
    const uint32_t code = b[p8_tile_off(c, h, pos % c.block_size) + o];
    // (the conversion yields a pair; a code is exact in bf16, and so is its product with the scale)
    const auto v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code, p8_scale(b[p8_scale_off(c, h) + kv]), false);
    return bf16_to_f32(__builtin_bit_cast(uint32_t, v) & 0xffff);
}

int p8_check(const dkv_paged8_t* c, int layer, const char* fn);
int p8_check_hot(const dkv_paged8_t& c, int T, const char* fn);

}  // namespace dkv
