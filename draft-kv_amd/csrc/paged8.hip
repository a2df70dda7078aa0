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
    if (c->n_kv_heads > 65535 || c->batch > 65535) return fail(DKV_EINVAL, f + ": too many heads or sequences");
    if (reinterpret_cast<uintptr_t>(c->pool) % 16 || reinterpret_cast<uintptr_t>(c->tail) % 16 ||
        reinterpret_cast<uintptr_t>(c->hot) % 16)
        return fail(DKV_EINVAL, f + ": pool, tail and hot must be 16-byte aligned");
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
// A workgroup owns one block of one (sequence, KV head): its bf16 tiles are put together in LDS (rows that were there
// from the ring, new ones from the inputs, zeros past the end), go to the ring or to hot in 16-byte pieces, and, where
// the block is now full, are coded: one maximum over the block, then one conversion per value. K and V in turn share
// the buffer. The inputs are read once; what is written is the codes, or the rows, or both.
constexpr int AP_THREADS = 256;

__device__ __forceinline__ uint32_t p8_biased_exponent(uint32_t amax_bits) {
    // amax: the bf16 magnitude of the block's largest finite value. Its exponent field x and mantissa m (7 bits):
    // amax = (1 + m / 128) 2^(x - 127), and 448 = 1.75 * 2^8
    if (amax_bits == 0) return 127;
    const int x = amax_bits >> 7, m = amax_bits & 0x7f;
    const int e = x - 127 - 8 + (m > 96 ? 1 : 0);   // (x = 0, subnormal: the clamp)
    return min(max(e, -126), 119) + 127;            // 448 * 2^119 is the largest code that float32 and bf16 hold
}

template <class X>
__global__ void __launch_bounds__(AP_THREADS) paged8_append_kernel(dkv_paged8_t c, int layer, const X* __restrict__ k,
                                                                   const X* __restrict__ v, int T, bool in_ring,
                                                                   const int32_t* __restrict__ start,
                                                                   const int32_t* __restrict__ count) {
    const int h = blockIdx.y, s = blockIdx.z, D = c.head_dim, DP = p8_dp(D), bs = c.block_size, H = c.n_kv_heads;
    const int s0 = start[s], n = p8_new_rows(c, T, s0, count, s), end = s0 + n;
    const int base = s0 / bs * bs, p0 = base + blockIdx.x * bs;   // the block's first position
    if (n <= 0 || p0 >= end) return;
    const bool sealed = p0 + bs <= end;
    const int new0 = max(p0, s0), new1 = min(p0 + bs, end);
    // tiles to put together: all of the block where it is coded or moves to hot, else those with new rows
    const int t0 = sealed || !in_ring ? 0 : (new0 - p0) / 16, t1 = (new1 - p0 + 15) / 16;

    extern __shared__ __align__(16) uint32_t ap_lds[];
    uint32_t* red = ap_lds;                                                  // [AP_THREADS / WAVE]
    uint16_t* tile = reinterpret_cast<uint16_t*>(ap_lds + AP_THREADS / WAVE);   // [bs / 16][16 * DP]
    const int tid = threadIdx.x;
    uint8_t* block = sealed ? const_cast<uint8_t*>(p8_block(c, s, layer, p0)) : nullptr;
    for (int kv = 0; kv < 2; ++kv) {
        const X* x = kv ? v : k;
        const int pieces = 2 * DP;   // 16-byte pieces per bf16 tile
        for (int i = t0 * pieces + tid; i < t1 * pieces; i += AP_THREADS) {
            const int t = i / pieces, pc = i % pieces;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (p0 + 16 * t < s0)   // rows that were there
                w = reinterpret_cast<const uint4*>(p8_ring_tile(c, s, layer, h, p0 + 16 * t) + kv * 16 * DP)[pc];
            reinterpret_cast<uint4*>(tile)[i] = w;
        }
        __syncthreads();
        for (int i = tid; i < (new1 - new0) * D; i += AP_THREADS) {
            const int pos = new0 + i / D, d = i % D, o = pos - p0;
            const float f = p8_load(x, (((int64_t)s * T + (pos - s0)) * H + h) * D + d);
            tile[o / 16 * 16 * DP + (kv ? p8_v_off(DP, o % 16, d) : p8_k_off(DP, o % 16, d))] = f32_to_bf16_rne(f);
        }
        // (rows of the ring's tile past the end are stale)
        if (new1 % 16)
            for (int i = tid; i < (16 - new1 % 16) * DP; i += AP_THREADS) {
                const int o = new1 - p0 + i / DP, d = i % DP;
                tile[o / 16 * 16 * DP + (kv ? p8_v_off(DP, o % 16, d) : p8_k_off(DP, o % 16, d))] = 0;
            }
        __syncthreads();
        for (int i = t0 * pieces + tid; i < t1 * pieces; i += AP_THREADS) {
            const int pos = p0 + i / pieces * 16;
            uint16_t* to = (in_ring ? p8_ring_tile(c, s, layer, h, pos) : p8_hot_tile(c, s, h, pos, base)) + kv * 16 * DP;
            reinterpret_cast<uint4*>(to)[i % pieces] = reinterpret_cast<const uint4*>(tile)[i];
        }
        if (sealed) {   // uniform over the workgroup
            uint32_t mx = 0;
            for (int i = tid; i < bs * DP / 2; i += AP_THREADS) {
                const uint32_t w = reinterpret_cast<const uint32_t*>(tile)[i], a = w & 0x7fff, b = w >> 16 & 0x7fff;
                if (a < 0x7f80) mx = max(mx, a);
                if (b < 0x7f80) mx = max(mx, b);
            }
            for (int o = 32; o > 0; o >>= 1) mx = max(mx, (uint32_t)__shfl_xor((int)mx, o));
            if (tid % WAVE == 0) red[tid / WAVE] = mx;
            __syncthreads();
            for (int w = 0; w < AP_THREADS / WAVE; ++w) mx = max(mx, red[w]);
            const uint32_t e = p8_biased_exponent(mx);
            const float down = ldexpf(1.0f, 127 - (int)e);   // 2^-e, a normal number
            for (int i = tid; i < bs * DP / 8; i += AP_THREADS) {
                const uint4 w = reinterpret_cast<const uint4*>(tile)[i];
                auto pack = [&](uint32_t p, uint32_t q) {
                    float f[4] = {__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u), __uint_as_float(q << 16),
                                  __uint_as_float(q & 0xffff0000u)};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f[j] *= down;
                        // infinities become NaN; magnitudes past 448 * 2^119 saturate
                        f[j] = fabsf(f[j]) < INFINITY ? fminf(fmaxf(f[j], -448.0f), 448.0f) : __uint_as_float(0x7fc00000);
                    }
                    int r = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
                    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], r, true);
                };
                const int t = i / (2 * DP), pc = i % (2 * DP);
                uint8_t* to = block + p8_tile_off(c, h, 16 * t) + kv * 16 * DP;
                reinterpret_cast<uint2*>(to)[pc] = make_uint2(pack(w.x, w.y), pack(w.z, w.w));
            }
            if (tid == 0) block[p8_scale_off(c, h) + kv] = (uint8_t)e;
        }
        __syncthreads();   // the buffer and red are free again
    }
}

// After an append through hot: the last tail_rows rows of the sequence, whole tiles, into the ring.
__global__ void __launch_bounds__(AP_THREADS) paged8_tail_kernel(dkv_paged8_t c, int layer, int T,
                                                                 const int32_t* __restrict__ start,
                                                                 const int32_t* __restrict__ count) {
    const int h = blockIdx.y, s = blockIdx.z, s0 = start[s], n = p8_new_rows(c, T, s0, count, s), end = s0 + n;
    const int base = s0 / c.block_size * c.block_size, pos = ((end + 15) / 16 - 1 - (int)blockIdx.x) * 16;
    if (n <= 0 || pos < base) return;
    const uint4* from = reinterpret_cast<const uint4*>(p8_hot_tile(c, s, h, pos, base));
    uint4* to = reinterpret_cast<uint4*>(p8_ring_tile(c, s, layer, h, pos));
    for (int i = threadIdx.x; i < 4 * p8_dp(c.head_dim); i += AP_THREADS) to[i] = from[i];
}

__global__ void __launch_bounds__(256) paged8_read_kernel(dkv_paged8_t c, int layer, const int32_t* __restrict__ first,
                                                          const int32_t* __restrict__ length, int T,
                                                          float* __restrict__ k, float* __restrict__ v) {
    const int s = blockIdx.z, HD = c.n_kv_heads * c.head_dim, len = length[s];
    for (int t = blockIdx.y; t < T; t += gridDim.y) {
        const int64_t pos = (int64_t)first[s] + t;
        for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < HD; i += gridDim.x * blockDim.x) {
            const int h = i / c.head_dim, d = i % c.head_dim;
            const bool live = pos >= 0 && pos < len && pos < (int64_t)c.max_blocks * c.block_size;
            const int64_t o = ((int64_t)s * T + t) * HD + i;
            k[o] = live ? p8_value(c, s, layer, (int)pos, len, h, d, 0) : 0.0f;
            v[o] = live ? p8_value(c, s, layer, (int)pos, len, h, d, 1) : 0.0f;
        }
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
    const size_t lds = sizeof(uint32_t) * (AP_THREADS / WAVE) + (size_t)c.block_size * p8_dp(c.head_dim) * 2;
    static size_t done[2][16] = {};
    if (!reserve_lds(in_dtype == DKV_F32 ? reinterpret_cast<const void*>(paged8_append_kernel<float>)
                                         : reinterpret_cast<const void*>(paged8_append_kernel<uint16_t>),
                     lds, done[in_dtype == DKV_F32]))
        return fail(DKV_ELAUNCH, "dkv_paged8_append: cannot reserve " + std::to_string(lds) + " B of LDS");
    const dim3 grid((T + c.block_size - 2) / c.block_size + 1, c.n_kv_heads, c.batch), blk(AP_THREADS);
    hipStream_t st = as_stream(stream);
    if (in_dtype == DKV_F32)
        hipLaunchKernelGGL((paged8_append_kernel<float>), grid, blk, lds, st, c, layer, static_cast<const float*>(k),
                           static_cast<const float*>(v), T, in_ring, start, count);
    else
        hipLaunchKernelGGL((paged8_append_kernel<uint16_t>), grid, blk, lds, st, c, layer,
                           static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), T, in_ring, start, count);
    if ((rc = check_launch("dkv_paged8_append"))) return rc;
    if (in_ring) return DKV_OK;
    hipLaunchKernelGGL(paged8_tail_kernel, dim3(c.tail_rows / 16, c.n_kv_heads, c.batch), blk, 0, st, c, layer, T, start,
                       count);
    return check_launch("dkv_paged8_append(tail)");
}

extern "C" int dkv_paged8_read(const dkv_paged8_t* cache, int32_t layer, const int32_t* first, const int32_t* length,
                               int32_t T, float* k, float* v, dkv_stream_t stream) {
    using namespace dkv;
    const int rc = p8_check(cache, layer, "dkv_paged8_read");
    if (rc) return rc;
    DKV_REQUIRE(first && length && k && v, "dkv_paged8_read: NULL argument");
    if (T <= 0) return DKV_OK;
    const int HD = cache->n_kv_heads * cache->head_dim;
    hipLaunchKernelGGL(paged8_read_kernel, dim3((HD + 255) / 256, std::min(T, 65535), cache->batch), dim3(256), 0,
                       as_stream(stream), *cache, layer, first, length, T, k, v);
    return check_launch("dkv_paged8_read");
}
