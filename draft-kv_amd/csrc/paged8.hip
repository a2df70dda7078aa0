// The full cache in 8 bits: append and read. (Layout and definition: paged8.h; attention: paged8_attn.hip.)
// Reference: draftkv/paged.py:76-176, whose cache is float32.
#include <algorithm>

#include "paged8.h"

namespace dkv {

int p8_check(const dkv_paged8_t* c, int layer, const char* fn) {
    const std::string f = fn;
    if (!c || !c->pool || !c->block_table || !c->tail) return fail(DKV_EINVAL, f + ": NULL cache");
    if (c->batch < 1 || c->n_layers < 1 || c->n_kv_heads < 1 || c->max_blocks < 1)
        return fail(DKV_EINVAL, f + ": bad cache shape");
    if (c->head_dim < 1 || c->head_dim > P8_MAXD) return fail(DKV_EINVAL, f + ": head_dim must be 1..256");
    if (c->block_size != 16 && c->block_size != 32 && c->block_size != 64 && c->block_size != 128)
        return fail(DKV_EINVAL, f + ": block_size must be 16, 32, 64 or 128");
    if (c->tail_rows % 16 || c->tail_rows < c->block_size + 16)
        return fail(DKV_EINVAL, f + ": tail_rows must be a multiple of 16, at least block_size + 16");
    if (layer < 0 || layer >= c->n_layers) return fail(DKV_EINVAL, f + ": layer out of range");
    if (c->n_kv_heads > 32767 || c->batch > 65535) return fail(DKV_EINVAL, f + ": too many heads or sequences");
    if (reinterpret_cast<uintptr_t>(c->pool) % 16 || reinterpret_cast<uintptr_t>(c->tail) % 16 ||
        reinterpret_cast<uintptr_t>(c->hot) % 16 || reinterpret_cast<uintptr_t>(c->held) % 16)
        return fail(DKV_EINVAL, f + ": pool, tail, hot and held must be 16-byte aligned");
    return DKV_OK;
}

// A call's rows must lie in the ring beside the open block, or in hot.
int p8_check_hot(const dkv_paged8_t& c, int T, const char* fn) {
    const int need = p8_hot_rows(c, T);
    if (need && (!c.hot || c.hot_rows < need || c.hot_rows % 16))
        return fail(DKV_EWORKSPACE, std::string(fn) + ": " + std::to_string(T) + " rows need hot rows (" +
                                        std::to_string(need) + ", a multiple of 16)");
    return DKV_OK;
}

// ---------------------------------------------------------------- append
// A workgroup owns one block of one (sequence, KV head, K or V); a wave, panels of its tiles: lane 16 q + c takes the
// values that it stores (K: PB channels of a token; V: four tokens of PB / 4 channels), so nothing is transposed and the
// rows stay in registers from the load to the codes. They go to the ring or to hot as bf16 and, where the block is now
// full, into codes: one maximum over the block, then a conversion per pair. The inputs are read once; rows that the
// block held before come from the ring, or from held, and go back to the ring where this append leaves them room. Bound
// by that traffic for a prompt (4096 tokens, 8 heads of 128, float32 in, 59 MB: 19 us, 3.1 TB/s), by the latency of a
// load and a store for single tokens.
constexpr int AP_WAVES = 8;

__device__ __forceinline__ uint32_t p8_biased_exponent(uint32_t amax_bits) {
    // amax: the bf16 magnitude of the block's largest finite value. Its exponent field x and mantissa m (7 bits):
    // amax = (1 + m / 128) 2^(x - 127), and 448 = 1.75 * 2^8
    if (amax_bits == 0) return 127;
    const int x = amax_bits >> 7, m = amax_bits & 0x7f;
    const int e = x - 127 - 8 + (m > 96 ? 1 : 0);   // (x = 0, subnormal: the clamp)
    return min(max(e, -126), 119) + 127;            // 448 * 2^119 is the largest code that float32 and bf16 hold
}

__device__ __forceinline__ uint32_t ap_bits(const float* p) { return f32_to_bf16_rne(*p); }
__device__ __forceinline__ uint32_t ap_bits(const uint16_t* p) { return *p; }
// N values from p on as bf16 pairs, 16 bytes at a time
template <int N>
__device__ __forceinline__ void ap_row(const float* p, uint32_t* r) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const float4 f = reinterpret_cast<const float4*>(p)[i];
        r[2 * i] = f32_to_bf16_rne(f.x) | (uint32_t)f32_to_bf16_rne(f.y) << 16;
        r[2 * i + 1] = f32_to_bf16_rne(f.z) | (uint32_t)f32_to_bf16_rne(f.w) << 16;
    }
}
template <int N>
__device__ __forceinline__ void ap_row(const uint16_t* p, uint32_t* r) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) reinterpret_cast<uint4*>(r)[i] = reinterpret_cast<const uint4*>(p)[i];
}

// What a workgroup's lanes know of their rows. PB: values per lane and panel; VEC: a lane's PB channels of K lie within
// D and are 16-byte aligned in the input.
template <class X, bool VEC, int PB>
struct ApRows {
    const X* x;        // row 0 of the call, this head
    int64_t ld;        // values from row to row
    int s0, end, D, kv, col, q;

    // panel i of the tile at pos; ring: that tile's panel in the ring, read for rows before s0
    __device__ __forceinline__ void load(int pos, int i, const uint16_t* ring, uint32_t (&r)[PB / 2]) const {
        constexpr int PW = 4 * PB;
#pragma unroll
        for (int e = 0; e < PB / 2; ++e) r[e] = 0;   // rows past the end, channels past D
        const int lane = 16 * q + col;
        if (kv == 0) {
            const int row = pos + col, d0 = PW * i + PB * q;
            if (row < s0) {
#pragma unroll
                for (int e = 0; e < PB / 8; ++e) reinterpret_cast<uint4*>(r)[e] = reinterpret_cast<const uint4*>(ring + lane * PB)[e];
            } else if (row < end) {
                const X* p = x + (row - s0) * ld + d0;
                if constexpr (VEC) {
                    if (d0 < D) ap_row<PB>(p, r);
                } else {
#pragma unroll
                    for (int e = 0; e < PB; ++e)
                        if (d0 + e < D) r[e / 2] |= ap_bits(p + e) << 16 * (e & 1);
                }
            }
            return;
        }
        const int row = pos + 4 * q, d0 = PW * i + col;
        uint32_t old[PB / 2];
        if (row < s0) {
#pragma unroll
            for (int e = 0; e < PB / 8; ++e) reinterpret_cast<uint4*>(old)[e] = reinterpret_cast<const uint4*>(ring + lane * PB)[e];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (row + j < s0) {
#pragma unroll
                for (int t = 0; t < PB / 4; ++t) r[2 * t + j / 2] |= old[2 * t + j / 2] & 0xffffu << 16 * (j & 1);
            } else if (row + j < end) {
                const X* p = x + (row + j - s0) * ld + d0;
#pragma unroll
                for (int t = 0; t < PB / 4; ++t)
                    if (d0 + 16 * t < D) r[2 * t + j / 2] |= ap_bits(p + 16 * t) << 16 * (j & 1);
            }
        }
    }
};

template <class X, bool VEC, int PB>
__global__ void __launch_bounds__(64 * AP_WAVES, 8) paged8_append_kernel(dkv_paged8_t c, int layer, const X* __restrict__ k,
                                                                      const X* __restrict__ v, int T, bool in_ring,
                                                                      const int32_t* __restrict__ start,
                                                                      const int32_t* __restrict__ count) {
    constexpr int PW = 4 * PB, UNITS = 4;   // panels per wave: 8 tiles of 4 panels over 8 waves
    const int h = blockIdx.y >> 1, kv = blockIdx.y & 1, s = blockIdx.z, D = c.head_dim, DP = p8_dp(D), bs = c.block_size;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE, waves = blockDim.x / WAVE;
    const int panels = DP / PW;   // unit u: panel u % panels of tile u / panels; a wave has the units wave + x * waves
    int tag = -1;                 // lane x: the first block's tag of unit x
    if (c.held && blockIdx.x == 0 && lane < UNITS && wave + lane * waves < bs / 16 * panels) {
        const int u = wave + lane * waves;
        tag = *p8_held_tag(c, s, layer, h, u / panels * 16, kv, u % panels);
    }
    const int s0 = start[s], n = p8_new_rows(c, T, s0, count, s), end = s0 + n;
    const int base = s0 / bs * bs, p0 = base + blockIdx.x * bs;   // the block's first position
    if (n <= 0 || p0 >= end) return;
    const bool sealed = p0 + bs <= end;
    const int new0 = max(p0, s0), new1 = min(p0 + bs, end);
    // tiles to put together: all of the block where it is coded or moves to hot, else those with new rows
    const int t0 = sealed || !in_ring ? 0 : (new0 - p0) / 16, t1 = (new1 - p0 + 15) / 16;
    // (looked up here: beside the loads of the rows, not behind them)
    uint8_t* block = sealed ? const_cast<uint8_t*>(p8_block(c, s, layer, p0)) : nullptr;
    const ApRows<X, VEC, PB> rows{(kv ? v : k) + ((int64_t)s * T * c.n_kv_heads + h) * D, (int64_t)c.n_kv_heads * D,
                                  s0, end, D, kv, lane % 16, lane / 16};
    auto at = [&](uint16_t* tile, int i) { return tile + kv * 16 * DP + i * 16 * PW; };
    auto put = [&](uint16_t* to, const uint32_t(&r)[PB / 2]) {
#pragma unroll
        for (int e = 0; e < PB / 8; ++e) reinterpret_cast<uint4*>(to + lane * PB)[e] = reinterpret_cast<const uint4*>(r)[e];
    };
    const int last = (end - 1) / 16 * 16;                       // the last tile
    const int held = (s0 - base + 15) / 16 * 16;                // rows of the tiles that the first block reads in the ring
    // Where held has a tile of the first block (rarely), it goes back to the ring, whose place nothing else touches. A tag
    // of a later block is void, the sequence was cut before it: an append that goes on from here to that block has all
    // the tiles of its first block here.
    if (__any(tag >= base + bs || (tag >= base && tag < p0 + 16 * t1))) {
        for (int x = 0; x < UNITS; ++x) {
            const int u = wave + x * waves, i = u % panels, pos = p0 + 16 * (u / panels), was = __shfl(tag, x);
            if (u >= t1 * panels) break;
            if (was != pos && was < base + bs) continue;
            if (lane == 0) *p8_held_tag(c, s, layer, h, pos, kv, i) = -1;
            if (was != pos || pos >= s0) continue;
            const uint16_t* from = at(p8_held_tile(c, s, layer, h, pos), i) + lane * PB;
            uint16_t* to = at(p8_ring_tile(c, s, layer, h, pos), i) + lane * PB;
#pragma unroll
            for (int e = 0; e < PB / 8; ++e) reinterpret_cast<uint4*>(to)[e] = reinterpret_cast<const uint4*>(from)[e];
        }
    }
    __align__(16) uint32_t r[UNITS][PB / 2];
#pragma unroll
    for (int x = 0; x < UNITS; ++x) {
        const int u = wave + x * waves, t = u / panels, i = u % panels, pos = p0 + 16 * t;
        if (t >= t0 && t < t1) rows.load(pos, i, at(p8_ring_tile(c, s, layer, h, pos), i), r[x]);
    }
#pragma unroll
    for (int x = 0; x < UNITS; ++x) {
        const int u = wave + x * waves, t = u / panels, i = u % panels, pos = p0 + 16 * t;
        if (t >= t1) break;
        if (t < t0) continue;
        if (!in_ring) put(at(p8_hot_tile(c, s, h, pos, base), i), r[x]);
        // the ring keeps the last tail_rows rows. A tile whose place there holds rows that the first block still
        // reads is left to the wave that reads them
        if (last - pos < c.tail_rows && (pos - base < c.tail_rows || (pos - base) % c.tail_rows >= held))
            put(at(p8_ring_tile(c, s, layer, h, pos), i), r[x]);
        if (!in_ring && pos < s0) {
            const int later = last - (last - pos) % c.tail_rows;
            if (later != pos) {
                __align__(16) uint32_t y[PB / 2];
                rows.load(later, i, nullptr, y);
                put(at(p8_ring_tile(c, s, layer, h, later), i), y);
                if (c.held) {
                    put(at(p8_held_tile(c, s, layer, h, pos), i), r[x]);
                    if (lane == 0) *p8_held_tag(c, s, layer, h, pos, kv, i) = pos;
                }
            }
        }
    }
    if (!sealed) return;   // uniform over the workgroup
    uint32_t mx = 0;
#pragma unroll
    for (int x = 0; x < UNITS; ++x)
        if ((wave + x * waves) / panels < t1) {
#pragma unroll
            for (int e = 0; e < PB / 2; ++e) {
                const uint32_t a = r[x][e] & 0x7fff, b = r[x][e] >> 16 & 0x7fff;
                if (a < 0x7f80) mx = max(mx, a);
                if (b < 0x7f80) mx = max(mx, b);
            }
        }
    for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o));
    __shared__ uint32_t red[AP_WAVES];
    if (lane == 0) red[wave] = mx;
    __syncthreads();
    for (int w = 0; w < waves; ++w) mx = max(mx, red[w]);
    const uint32_t e = p8_biased_exponent(mx);
    const float down = ldexpf(1.0f, 127 - (int)e);   // 2^-e, a normal number
    auto pack = [&](uint32_t p, uint32_t q) {
        float f[4] = {__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u), __uint_as_float(q << 16),
                      __uint_as_float(q & 0xffff0000u)};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] *= down;
            // infinities become NaN; magnitudes past 448 * 2^119 saturate
            f[j] = fabsf(f[j]) < INFINITY ? fminf(fmaxf(f[j], -448.0f), 448.0f) : __uint_as_float(0x7fc00000);
        }
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
    };
#pragma unroll
    for (int x = 0; x < UNITS; ++x) {
        const int u = wave + x * waves, t = u / panels, i = u % panels;
        if (t >= t1) break;
        uint2* to = reinterpret_cast<uint2*>(block + p8_tile_off(c, h, 16 * t) + kv * 16 * DP + i * 16 * PW + lane * PB);
#pragma unroll
        for (int o = 0; o < PB / 8; ++o)
            to[o] = make_uint2(pack(r[x][4 * o], r[x][4 * o + 1]), pack(r[x][4 * o + 2], r[x][4 * o + 3]));
    }
    if (threadIdx.x == 0) block[p8_scale_off(c, h) + kv] = (uint8_t)e;
}

// ---------------------------------------------------------------- read
// A workgroup takes one tile of one (head, K or V): a thread four values that lie together, channels of a token of K,
// tokens of a channel of V. Bound by the rows that it writes (4096 tokens, 8 heads of 128, 42 MB: 14 us).
__global__ void __launch_bounds__(256) paged8_read_kernel(dkv_paged8_t c, int layer, const int32_t* __restrict__ first,
                                                          const int32_t* __restrict__ length, int T,
                                                          float* __restrict__ k, float* __restrict__ v, bool vec) {
    const int h = blockIdx.y >> 1, kv = blockIdx.y & 1, s = blockIdx.z, D = c.head_dim, DP = p8_dp(D), H = c.n_kv_heads;
    const int64_t f0 = first[s], rows = (int64_t)c.max_blocks * c.block_size;
    const int64_t p0 = (f0 >> 4 << 4) + 16 * (int64_t)blockIdx.x;   // the tile's first position, before f0 for some
    const int64_t len = min((int64_t)length[s], rows);
    if (p0 >= f0 + T) return;
    float* out = (kv ? v : k) + ((int64_t)s * T * H + h) * D;   // + (pos - f0) * H * D + d
    const bool any = p0 >= 0 && p0 < len, ring = any && p0 >= length[s] / c.block_size * c.block_size;
    const uint16_t* tail = nullptr;
    const uint8_t* code = nullptr;
    float scale = 0.0f;
    if (ring) tail = p8_open_tile(c, s, layer, h, (int)p0) + kv * 16 * DP;
    else if (any) {
        const uint8_t* b = p8_block(c, s, layer, (int)p0);
        code = b + p8_tile_off(c, h, (int)(p0 % c.block_size)) + kv * 16 * DP;
        scale = p8_scale(b[p8_scale_off(c, h) + kv]);
    }
    for (int i = threadIdx.x; i < 4 * DP; i += 256) {
        const int token = kv ? i / DP * 4 : i / (DP / 4), d = kv ? i % DP : i % (DP / 4) * 4;
        if (d >= D) continue;
        const int o = kv ? p8_v_off(DP, token, d) : p8_k_off(DP, token, d);
        float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (ring) {
            const uint2 w = *reinterpret_cast<const uint2*>(tail + o);
            f[0] = bf16_to_f32(w.x & 0xffff), f[1] = bf16_to_f32(w.x >> 16), f[2] = bf16_to_f32(w.y & 0xffff), f[3] = bf16_to_f32(w.y >> 16);
        } else if (any) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(code + o);
            // (a code is exact in bf16, and so is its product with the scale)
            const uint32_t a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
            const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true));
            f[0] = bf16_to_f32(a & 0xffff), f[1] = bf16_to_f32(a >> 16), f[2] = bf16_to_f32(b & 0xffff), f[3] = bf16_to_f32(b >> 16);
        }
        if (kv) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t pos = p0 + token + j;
                if (pos >= f0 && pos < f0 + T) out[(pos - f0) * H * D + d] = pos < len ? f[j] : 0.0f;
            }
            continue;
        }
        const int64_t pos = p0 + token;
        if (pos < f0 || pos >= f0 + T) continue;
        float* to = out + (pos - f0) * H * D + d;
        const bool live = pos < len;
        if (vec) *reinterpret_cast<float4*>(to) = live ? make_float4(f[0], f[1], f[2], f[3]) : make_float4(0, 0, 0, 0);
        else
            for (int e = 0; e < 4 && d + e < D; ++e) to[e] = live ? f[e] : 0.0f;
    }
}

}  // namespace dkv

extern "C" int64_t dkv_paged8_block_bytes(int32_t n_kv_heads, int32_t head_dim, int32_t block_size) {
    return n_kv_heads < 1 || head_dim < 1 || block_size < 1 ? 0 : dkv::p8_block_bytes(n_kv_heads, head_dim, block_size);
}

extern "C" int64_t dkv_paged8_row_bytes(int32_t n_kv_heads, int32_t head_dim) {
    return n_kv_heads < 1 || head_dim < 1 ? 0 : dkv::p8_row_bytes(n_kv_heads, head_dim);
}

extern "C" int32_t dkv_paged8_hot_rows(const dkv_paged8_t* cache, int32_t T) {
    return !cache || T < 1 ? 0 : dkv::p8_hot_rows(*cache, T);
}

extern "C" int64_t dkv_paged8_held_bytes(const dkv_paged8_t* cache) {
    using namespace dkv;
    if (!cache || cache->batch < 1 || cache->n_layers < 1 || cache->n_kv_heads < 1 || cache->head_dim < 1 || cache->block_size < 16) return 0;
    return (int64_t)cache->batch * cache->n_layers * cache->n_kv_heads * (cache->block_size / 16) * p8_held_stride(p8_dp(cache->head_dim));
}

extern "C" int dkv_paged8_append(const dkv_paged8_t* cache, int32_t layer, const void* k, const void* v,
                                 int32_t in_dtype, int32_t T, const int32_t* start, const int32_t* count,
                                 dkv_stream_t stream) {
    using namespace dkv;
    int rc = p8_check(cache, layer, "dkv_paged8_append");
    if (rc) return rc;
    DKV_REQUIRE(k && v && start, "dkv_paged8_append: NULL argument");
    DKV_REQUIRE(in_dtype == DKV_F32 || in_dtype == DKV_BF16, "dkv_paged8_append: bad input dtype");
    DKV_REQUIRE(T <= 1 << 24, "dkv_paged8_append: too many rows");
    if (T <= 0) return DKV_OK;
    const dkv_paged8_t c = *cache;
    if ((rc = p8_check_hot(c, T, "dkv_paged8_append"))) return rc;
    const bool in_ring = p8_in_ring(c, T);
    // a lane's channels of K: whole 16-byte pieces, all or none of them past D
    const int pb = c.head_dim <= 32 ? 8 : 16, units = c.block_size / 16 * (p8_dp(c.head_dim) / (4 * pb));
    const bool vec = c.head_dim % pb == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0;
    const dim3 grid((T + c.block_size - 2) / c.block_size + 1, 2 * c.n_kv_heads, c.batch), blk(WAVE * std::min(AP_WAVES, units));
    hipStream_t st = as_stream(stream);
#define DKV_P8A(XX, VV, BB)                                                                                               \
    hipLaunchKernelGGL((paged8_append_kernel<XX, VV, BB>), grid, blk, 0, st, c, layer, static_cast<const XX*>(k),          \
                       static_cast<const XX*>(v), T, in_ring, start, count)
#define DKV_P8B(XX)                           \
    if (pb == 8 && vec) DKV_P8A(XX, true, 8); \
    else if (pb == 8) DKV_P8A(XX, false, 8);  \
    else if (vec) DKV_P8A(XX, true, 16);      \
    else DKV_P8A(XX, false, 16)
    if (in_dtype == DKV_F32) {
        DKV_P8B(float);
    } else {
        DKV_P8B(uint16_t);
    }
#undef DKV_P8B
#undef DKV_P8A
    return check_launch("dkv_paged8_append");
}

extern "C" int dkv_paged8_read(const dkv_paged8_t* cache, int32_t layer, const int32_t* first, const int32_t* length,
                               int32_t T, float* k, float* v, dkv_stream_t stream) {
    using namespace dkv;
    const int rc = p8_check(cache, layer, "dkv_paged8_read");
    if (rc) return rc;
    DKV_REQUIRE(first && length && k && v, "dkv_paged8_read: NULL argument");
    if (T <= 0) return DKV_OK;
    const bool vec = cache->head_dim % 4 == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0;
    hipLaunchKernelGGL(paged8_read_kernel, dim3((unsigned)(((int64_t)T + 30) / 16), 2 * cache->n_kv_heads, cache->batch), dim3(256), 0,
                       as_stream(stream), *cache, layer, first, length, T, k, v, vec);
    return check_launch("dkv_paged8_read");
}
