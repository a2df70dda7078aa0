// Microscaled 4-bit floating point (OCP MX 1.0, MXFP4): quantization, and the products of the model forwards with
// weights held in it. Reference: the `x @ W` products of model.py:113-133, gpt2.py:191-213, llama.py:187-225 (numpy
// float32 there).
//
// Format. Of every 32 values along k: a = max |x|, e = floor(log2 a) - 2 (0 where a = 0, at least -126), codes
// e2m1(x * 2^-e), nearest even, saturating at 6; a block with a NaN or an infinity has the NaN scale. The scale byte
// is e + 127.
//
// Layout, of weights and of quantized rows alike: tiles of 16 rows x 128 k, 1 KB, a row fragment's tiles consecutive
// along k. Lane 16 q + c of a tile holds row c, the block k = 32 q .. 32 q + 31: 16 bytes, two values a byte, the lower
// k in the low half. That is the operand of v_mfma_scale_f32_16x16x128_f8f6f4 as it is, and, word j converted to bf16,
// that of step j of four v_mfma_f32_16x16x32_bf16 (k = 32 q + 8 j + 0 .. 7 in both operands). The scale bytes of four
// tiles share a word per lane, which the matrix instruction selects from. Rows past the last are zeros, and so are
// columns past K.
//
// Arithmetic. K is cut into S chunks of whole tiles, S a function of (N, K) only; a chunk is one chain of matrix
// instructions in order, the chunks' sums are added in order, the bias last. A row's result is the same for any M.
#include <algorithm>
#include <initializer_list>

#include "dkv_common.h"

namespace dkv {

typedef __bf16 mx_bf16x8 __attribute__((ext_vector_type(8)));
typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef float mx_f32x2 __attribute__((ext_vector_type(2)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4)));

__host__ __device__ inline int64_t mx_frags(int64_t rows) { return (rows + 15) / 16; }
__host__ __device__ inline int64_t mx_tiles(int64_t k) { return (k + 127) / 128; }
__host__ __device__ inline int64_t mx_quads(int64_t k) { return (k + 511) / 512; }

constexpr int MX_NAN = 255;

// ---------------------------------------------------------------- quantize
// A workgroup takes 16 rows x 512 k: four tiles and their scale words. Four lanes share a block, a wave reads 512
// consecutive values of one row. Bound by the read of x.
template <class X>
__device__ __forceinline__ float mx_load(const X* p);
template <>
__device__ __forceinline__ float mx_load(const float* p) { return *p; }
template <>
__device__ __forceinline__ float mx_load(const uint16_t* p) { return bf16_to_f32(*p); }

template <class X>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(const X* __restrict__ x, int rows, int K, uint8_t* __restrict__ codes,
                                                           uint32_t* __restrict__ scales, float* __restrict__ values) {
    __shared__ __align__(16) uint32_t sc[16 * 4];   // [q][c] words of four tiles
    const int64_t quads = mx_quads(K), tiles = mx_tiles(K);
    const int64_t f = blockIdx.x / quads, quad = blockIdx.x % quads;
    const int tid = threadIdx.x, sub = tid % 4, b = tid % 64 / 4;   // block b of the 16 of the row's 512 k
    const int64_t k0 = quad * 512 + 32 * b + 8 * sub;
    const int64_t tile = quad * 4 + b / 4;
    for (int c = tid / 64; c < 16; c += 4) {
        const int64_t r = f * 16 + c;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = r < rows && k0 + i < K ? mx_load(x + r * K + k0 + i) : 0.0f;
        uint32_t a = 0;   // magnitudes order as their bits do; NaN and infinity come out largest
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(v[i]) & 0x7fffffffu);
        a = max(a, (uint32_t)__shfl_xor((int)a, 1));
        a = max(a, (uint32_t)__shfl_xor((int)a, 2));
        const int ex = a >> 23;
        const uint32_t s = a == 0 ? 127u : ex == 255 ? (uint32_t)MX_NAN : (uint32_t)max(ex - 2, 1);
        const float scale = __uint_as_float(s << 23);
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], scale, 3);
        if (tile < tiles)
            *reinterpret_cast<uint32_t*>(codes + (f * tiles + tile) * 1024 + (b % 4 * 16 + c) * 16 + 4 * sub) = w;
        if (sub == 0) reinterpret_cast<uint8_t*>(sc)[(b % 4 * 16 + c) * 4 + b / 4] = (uint8_t)s;
        if (values && r < rows) {
            const mx_f32x2 o[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1),
                                   __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3)};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k0 + i < K) values[r * K + k0 + i] = o[i / 2][i % 2];
        }
    }
    __syncthreads();
    if (tid < 64) scales[(f * quads + quad) * 64 + tid] = sc[tid];
}

__global__ void __launch_bounds__(256) mx4_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows,
                                                         int K, float* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)rows * K;
    if (i >= n) return;
    const int64_t r = i / K, k = i % K, f = r / 16, tile = k / 128;
    const int lane = (int)(k % 128 / 32 * 16 + r % 16);
    const uint32_t byte = codes[(f * mx_tiles(K) + tile) * 1024 + lane * 16 + k % 32 / 2];
    const float scale = __uint_as_float((uint32_t)scales[((f * mx_quads(K) + tile / 4) * 64 + lane) * 4 + tile % 4] << 23);
    const mx_f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(byte, scale, 0);
    out[i] = k % 2 ? v[1] : v[0];
}

// ---------------------------------------------------------------- product
struct MxArgs {
    const void* x;             // [M][K] float32 or bf16, or codes
    const uint32_t* xs;        // scale words of codes
    const uint8_t* w;
    const uint32_t* ws;
    const void* bias;          // [N] or null
    int bias_f32, y_f32, swiglu, vec;   // vec: rows of x are 16-byte aligned in whole runs of 8
    int M, N, K, tiles, quads;
    int S, CT;                 // chunks, tiles per chunk
    void* y;
};

// K chunks of a weight: enough for about a thousand waves at one row fragment each, of at least four tiles
__host__ inline void mx_chunks(int N, int K, int& S, int& CT) {
    const int tiles = (int)mx_tiles(K);
    S = std::min(8, (16384 + N - 1) / N);
    CT = std::max((tiles + S - 1) / S, std::min(4, tiles));
    S = (tiles + CT - 1) / CT;
}

__device__ __forceinline__ uint32_t mx_pair(uint32_t w, float scale, int j) {
    switch (j) {   // (the selector is an immediate)
        case 0: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
        case 1: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
        case 2: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
        default: return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    }
}
// eight codes as bf16 values
__device__ __forceinline__ mx_bf16x8 mx_operand(uint32_t w, float scale) {
    return __builtin_bit_cast(mx_bf16x8, mx_u32x4{mx_pair(w, scale, 0), mx_pair(w, scale, 1), mx_pair(w, scale, 2), mx_pair(w, scale, 3)});
}
__device__ __forceinline__ uint32_t mx_bf16_pair(float a, float b) {
    const __bf16 x = (__bf16)a, y = (__bf16)b;
    return (uint32_t)__builtin_bit_cast(uint16_t, x) | (uint32_t)__builtin_bit_cast(uint16_t, y) << 16;
}

// 8 values of row r of x from k on, as bf16 (zeros past K)
template <bool F32>
__device__ __forceinline__ mx_bf16x8 mx_x8(const MxArgs& A, int64_t r, int k) {
    const int64_t at = r * A.K + k;
    float v[8];
    if (A.vec) {
        if (k >= A.K) return __builtin_bit_cast(mx_bf16x8, mx_u32x4{0, 0, 0, 0});
        if constexpr (!F32) return __builtin_bit_cast(mx_bf16x8, *reinterpret_cast<const mx_u32x4*>(static_cast<const uint16_t*>(A.x) + at));
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(A.x) + at);
        const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(A.x) + at + 4);
        return __builtin_bit_cast(mx_bf16x8, mx_u32x4{mx_bf16_pair(a.x, a.y), mx_bf16_pair(a.z, a.w), mx_bf16_pair(b.x, b.y), mx_bf16_pair(b.z, b.w)});
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        v[i] = k + i >= A.K ? 0.0f : F32 ? static_cast<const float*>(A.x)[at + i] : bf16_to_f32(static_cast<const uint16_t*>(A.x)[at + i]);
    return __builtin_bit_cast(mx_bf16x8, mx_u32x4{mx_bf16_pair(v[0], v[1]), mx_bf16_pair(v[2], v[3]), mx_bf16_pair(v[4], v[5]), mx_bf16_pair(v[6], v[7])});
}

// outputs (m, n .. n + 3), n a multiple of 4
__device__ __forceinline__ void mx_store(const MxArgs& A, int64_t m, int n, mx_f32x4 t) {
    if (n >= A.N) return;   // the last fragment's rows past N
    if (A.swiglu) {   // rows of W interleave (gate, up); N is even
        for (int e = 0; e < 4; e += 2)
            if (n + e < A.N) {
                const float o = t[e] / (1.0f + __expf(-t[e])) * t[e + 1];
                const int64_t at = m * (A.N / 2) + (n + e) / 2;
                if (A.y_f32) static_cast<float*>(A.y)[at] = o;
                else static_cast<uint16_t*>(A.y)[at] = f32_to_bf16_rne(o);
            }
        return;
    }
    if (A.bias)
        for (int e = 0; e < 4; ++e)
            if (n + e < A.N) t[e] += load_elem(A.bias, n + e, A.bias_f32 ? DKV_F32 : DKV_BF16);
    const int64_t at = m * A.N + n;
    if (A.N % 4 == 0) {
        if (A.y_f32) *reinterpret_cast<mx_f32x4*>(static_cast<float*>(A.y) + at) = t;
        else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(A.y) + at) = make_uint2(mx_bf16_pair(t[0], t[1]), mx_bf16_pair(t[2], t[3]));
        return;
    }
    for (int e = 0; e < 4; ++e)
        if (n + e < A.N) {
            if (A.y_f32) static_cast<float*>(A.y)[at + e] = t[e];
            else static_cast<uint16_t*>(A.y)[at + e] = f32_to_bf16_rne(t[e]);
        }
}

enum { MX_XF32, MX_XBF16, MX_XMX4 };

// tile b of four of the 4-bit product: the scale bytes are selected by the instruction
__device__ __forceinline__ mx_f32x4 mx_mfma4(mx_i32x8 w, mx_i32x8 x, mx_f32x4 c, int b, uint32_t sw, uint32_t sx) {
    switch (b) {
        case 0: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, 4, 0, (int)sw, 0, (int)sx);
        case 1: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, 4, 1, (int)sw, 1, (int)sx);
        case 2: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, 4, 2, (int)sw, 2, (int)sx);
        default: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, c, 4, 4, 3, (int)sw, 3, (int)sx);
    }
}

// Grid (row fragment of W, group of MB 16-row tiles of x). One wave per chunk; the sums meet in LDS.
template <int XM, int MB>
__global__ void __launch_bounds__(512) mx4_gemm_kernel(MxArgs A) {
#pragma clang fp contract(off)
    extern __shared__ __align__(16) mx_f32x4 mx_lds[];   // [S][MB][64]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int col = lane % 16, q = lane / 16;
    const int64_t f = blockIdx.x, m0 = (int64_t)blockIdx.y * 16 * MB;
    const int t0 = wave * A.CT, t1 = min(t0 + A.CT, A.tiles);
    const mx_u32x4* wp = reinterpret_cast<const mx_u32x4*>(A.w + f * A.tiles * 1024) + lane;
    const uint32_t* wsp = A.ws + f * A.quads * 64 + lane;
    mx_f32x4 acc[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[i] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
    for (int t = t0; t < t1; ++t) {
        const mx_u32x4 w = wp[(int64_t)t * 64];
        const uint32_t sb = wsp[t / 4 * 64] >> 8 * (t % 4) & 0xff;
        if constexpr (XM == MX_XMX4) {
            const mx_i32x8 wv = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int64_t xf = min(m0 / 16 + i, mx_frags(A.M) - 1);
                const mx_u32x4 x = reinterpret_cast<const mx_u32x4*>(static_cast<const uint8_t*>(A.x) + (xf * A.tiles + t) * 1024)[lane];
                const uint32_t xb = A.xs[(xf * A.quads + t / 4) * 64 + lane] >> 8 * (t % 4) & 0xff;
                const mx_i32x8 xv = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
                acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, acc[i], 4, 4, 0, (int)sb, 0, (int)xb);
            }
        } else {
            const float scale = __uint_as_float(sb << 23);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const mx_bf16x8 wv = mx_operand(w[j], scale);
#pragma unroll
                for (int i = 0; i < MB; ++i) {
                    const int64_t r = min(m0 + 16 * i + col, (int64_t)A.M - 1);
                    const mx_bf16x8 xv = mx_x8<XM == MX_XF32>(A, r, 128 * t + 32 * q + 8 * j);
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv, acc[i], 0, 0, 0);
                }
            }
        }
    }
    if (A.S > 1) {
#pragma unroll
        for (int i = 0; i < MB; ++i) mx_lds[(wave * MB + i) * WAVE + lane] = acc[i];
        __syncthreads();
    }
    for (int i = wave; i < MB; i += A.S) {
        mx_f32x4 t;
        if (A.S > 1) {
            t = mx_lds[i * WAVE + lane];
            for (int s = 1; s < A.S; ++s) t += mx_lds[(s * MB + i) * WAVE + lane];
        } else {
            t = acc[0];
#pragma unroll
            for (int j = 1; j < MB; ++j)
                if (i == j) t = acc[j];
        }
        const int64_t m = m0 + 16 * i + col;
        if (m < A.M) mx_store(A, m, (int)f * 16 + 4 * q, t);
    }
}

// ---------------------------------------------------------------- product, many rows
// One workgroup: BN rows of W x BM rows of x, in steps of one tile (128 k). The order of the workgroups gives each XCD
// (workgroup g runs on XCD g % 8) one contiguous run of tiles, GM tiles of x by one of W at a time, so the 32 CUs of an
// XCD share both in its L2.
constexpr int MX_GM = 8;
__device__ __forceinline__ bool mx_tile_of(int mtiles, int ntiles, int& mt, int& nt) {
    const int groups = (mtiles + MX_GM - 1) / MX_GM, total = groups * MX_GM * ntiles, per = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= total) return false;
    const int grp = id / (MX_GM * ntiles), r = id % (MX_GM * ntiles);
    mt = grp * MX_GM + r % MX_GM, nt = r / MX_GM;
    return mt < mtiles;
}
__host__ inline unsigned mx_grid(int mtiles, int ntiles) {
    const int total = (mtiles + MX_GM - 1) / MX_GM * MX_GM * ntiles;
    return (unsigned)((total + 7) / 8 * 8);
}

// bf16 or float32 rows: four waves, NF fragments of W (16 NF rows) each, against the same 16 MB rows of x. W's codes go
// from memory to registers a tile ahead and are converted there (a conversion per two values, a ninth of the matrix
// instructions' time at NF x MB = 4 x 8); x goes through LDS, two stages. LDS holds x by rows of 16 pieces (8 values),
// piece p of row r in slot p ^ (r % 16): a row's pieces arrive together, and the 16 rows that an operand read takes lie
// on different banks. DMA: bf16 rows of whole tiles, straight to LDS; else through registers (rounding float32, zeros
// past K).
template <int XM, bool DMA, int NF, int MB, bool MULTI>
__global__ void __launch_bounds__(256, 2) mx4_tile_kernel(MxArgs A, int mtiles, int ntiles) {
#pragma clang fp contract(off)
    constexpr int BM = 16 * MB, STAGE = BM * 256;
    extern __shared__ __align__(16) char mx_smem[];   // [2][BM][16 slots] of 16 bytes
    int mt, nt;
    if (!mx_tile_of(mtiles, ntiles, mt, nt)) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE;
    const int col = lane % 16, q = lane / 16;
    const int64_t m0 = (int64_t)mt * BM;
    const int64_t frags = mx_frags(A.N), f0 = ((int64_t)nt * 4 + wave) * NF;
    const mx_u32x4* wp[NF];
    const uint32_t* sp[NF];
#pragma unroll
    for (int i = 0; i < NF; ++i) {
        const int64_t f = min(f0 + i, frags - 1);
        wp[i] = reinterpret_cast<const mx_u32x4*>(A.w + f * A.tiles * 1024) + lane;
        sp[i] = A.ws + f * A.quads * 64 + lane;
    }
    // x piece i of this thread: row 4 (wave + 4 i) + lane / 16, slot lane % 16
    auto x_row = [&](int i) { return 4 * (wave + 4 * i) + q; };
    auto x_at = [&](int i, int t) {   // its offset in x
        const int r = x_row(i);
        return min(m0 + r, (int64_t)A.M - 1) * A.K + 128 * t + 8 * (col ^ (r & 15));
    };
    auto dma = [&](int t) {
        const uint32_t base = lds_offset(mx_smem) + t % 2 * STAGE;
#pragma unroll
        for (int i = 0; i < MB; ++i)
            dma_b128<false>(A.x, (uint32_t)(2 * x_at(i, t)), base + (wave + 4 * i) * 1024);
    };
    constexpr int HALF = (MB + 1) / 2;   // pieces through registers at once
    mx_u32x4 xr[HALF];
    auto x_load = [&](int t, int h) {
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
            const int p = h * HALF + i;
            if (p >= MB) break;
            const int r = x_row(p), k = 128 * t + 8 * (col ^ (r & 15));
            xr[i] = __builtin_bit_cast(mx_u32x4, mx_x8<XM == MX_XF32>(A, min(m0 + r, (int64_t)A.M - 1), k));
        }
    };
    auto x_store = [&](int t, int h) {
#pragma unroll
        for (int i = 0; i < HALF; ++i) {
            const int p = h * HALF + i;
            if (p < MB) *reinterpret_cast<mx_u32x4*>(mx_smem + t % 2 * STAGE + (wave + 4 * p) * 1024 + 16 * lane) = xr[i];
        }
    };
    mx_f32x4 acc[NF][MB], tot[MULTI ? NF : 1][MULTI ? MB : 1];
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
    mx_u32x4 w[2][NF];
    uint32_t sc[NF], sn[NF];
    if constexpr (DMA) dma(0);
    else {
        x_load(0, 0);
        x_store(0, 0);
        x_load(0, 1);
        x_store(0, 1);
    }
#pragma unroll
    for (int i = 0; i < NF; ++i) {
        w[0][i] = *wp[i];
        sn[i] = *sp[i];
    }
    const int last = A.tiles - 1;
    int left = A.CT;
    for (int t0 = 0; t0 < A.tiles; t0 += 4) {
#pragma unroll
        for (int i = 0; i < NF; ++i) sc[i] = sn[i];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int t = t0 + b;
            if (t > last) break;   // uniform
            wait_loads_barrier<0>();   // stage t % 2 is there, and every wave is done with the other
            const int tn = min(t + 1, last);
            if constexpr (DMA) {
                if (t < last) dma(tn);
            } else {
                x_load(tn, 0);
            }
#pragma unroll
            for (int i = 0; i < NF; ++i) w[(b + 1) % 2][i] = wp[i][(int64_t)tn * 64];
            if (b == 0) {
                const int64_t qn = min(t0 / 4 + 1, A.quads - 1);
#pragma unroll
                for (int i = 0; i < NF; ++i) sn[i] = sp[i][qn * 64];
            }
            const char* xs = mx_smem + t % 2 * STAGE + col * 256;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!DMA && j == 2 && t < last) {
                    x_store(tn, 0);
                    x_load(tn, 1);
                }
                mx_bf16x8 wv[NF];
#pragma unroll
                for (int i = 0; i < NF; ++i) wv[i] = mx_operand(w[b % 2][i][j], __uint_as_float((sc[i] >> 8 * b & 0xff) << 23));
#pragma unroll
                for (int m = 0; m < MB; ++m) {
                    const mx_bf16x8 xv = *reinterpret_cast<const mx_bf16x8*>(xs + m * 4096 + ((4 * q + j) ^ col) * 16);
#pragma unroll
                    for (int i = 0; i < NF; ++i) acc[i][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[i], xv, acc[i][m], 0, 0, 0);
                }
            }
            if (!DMA && t < last) x_store(tn, 1);
            if constexpr (MULTI) {
                if (--left == 0 || t == last) {   // a chunk ends
                    const bool first = t < A.CT;
                    left = A.CT;
#pragma unroll
                    for (int i = 0; i < NF; ++i)
#pragma unroll
                        for (int m = 0; m < MB; ++m) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) tot[i][m][e] = first ? acc[i][m][e] : tot[i][m][e] + acc[i][m][e];
                            acc[i][m] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
                        }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int64_t r = m0 + 16 * m + col;
            if (r >= A.M || f0 + i >= frags) continue;
            mx_f32x4 o;
            if constexpr (MULTI) o = tot[i][m];
            else o = acc[i][m];
            mx_store(A, r, (int)(f0 + i) * 16 + 4 * q, o);
        }
}

// 4-bit rows: eight waves, four along W by two along x, 4 x MB fragments each. Both operands' tiles go to LDS as they
// are (1 KB, one load instruction each, two stages); the scale words straight to registers, once in four tiles. At
// 4 x 8 a tile of 256 x 256 reads 32 KB per 1024 cycles of matrix instructions, half of what an XCD's L2 gives its CUs.
template <int MB, bool MULTI>
__global__ void __launch_bounds__(512, 2) mx4_tile4_kernel(MxArgs A, int mtiles, int ntiles) {
#pragma clang fp contract(off)
    constexpr int NF = 4, WF = 4 * NF, XF = 2 * MB, STAGE = (WF + XF) * 1024, PER = (WF + XF) / 8;
    static_assert((WF + XF) % 8 == 0, "a stage's loads split evenly over the waves");
    extern __shared__ __align__(16) char mx_smem[];   // [2][W fragments, x fragments][1 KB]
    int mt, nt;
    if (!mx_tile_of(mtiles, ntiles, mt, nt)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int col = lane % 16, q = lane / 16, wn = wave % 4, wm = wave / 4;
    const int64_t frags = mx_frags(A.N), xfrags = mx_frags(A.M), f0 = (int64_t)nt * WF, x0 = (int64_t)mt * XF;
    const char* src[PER];   // this wave's fragments of a stage: wave, wave + 8, ...
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int p = wave + 8 * i;
        src[i] = p < WF ? reinterpret_cast<const char*>(A.w) + min(f0 + p, frags - 1) * A.tiles * 1024
                        : static_cast<const char*>(A.x) + min(x0 + (p - WF), xfrags - 1) * A.tiles * 1024;
    }
    auto dma = [&](int t) {
        const uint32_t base = lds_offset(mx_smem) + t % 2 * STAGE;
#pragma unroll
        for (int i = 0; i < PER; ++i) dma_b128<false>(src[i] + (int64_t)t * 1024, 16 * lane, base + (wave + 8 * i) * 1024);
    };
    const uint32_t *wsp[NF], *xsp[MB];
#pragma unroll
    for (int i = 0; i < NF; ++i) wsp[i] = A.ws + min(f0 + wn * NF + i, frags - 1) * A.quads * 64 + lane;
#pragma unroll
    for (int m = 0; m < MB; ++m) xsp[m] = A.xs + min(x0 + wm * MB + m, xfrags - 1) * A.quads * 64 + lane;
    mx_f32x4 acc[NF][MB], tot[MULTI ? NF : 1][MULTI ? MB : 1];
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
    uint32_t sw[NF], sx[MB], nw[NF], nx[MB];
    dma(0);
#pragma unroll
    for (int i = 0; i < NF; ++i) nw[i] = *wsp[i];
#pragma unroll
    for (int m = 0; m < MB; ++m) nx[m] = *xsp[m];
    const int last = A.tiles - 1;
    int left = A.CT;
    for (int t0 = 0; t0 < A.tiles; t0 += 4) {
#pragma unroll
        for (int i = 0; i < NF; ++i) sw[i] = nw[i];
#pragma unroll
        for (int m = 0; m < MB; ++m) sx[m] = nx[m];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int t = t0 + b;
            if (t > last) break;
            wait_loads_barrier<0>();
            if (t < last) dma(t + 1);
            if (b == 0) {
                const int64_t qn = min(t0 / 4 + 1, A.quads - 1);
#pragma unroll
                for (int i = 0; i < NF; ++i) nw[i] = wsp[i][qn * 64];
#pragma unroll
                for (int m = 0; m < MB; ++m) nx[m] = xsp[m][qn * 64];
            }
            const mx_u32x4* at = reinterpret_cast<const mx_u32x4*>(mx_smem + t % 2 * STAGE) + lane;
            mx_i32x8 wv[NF];
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                const mx_u32x4 v = at[(wn * NF + i) * WAVE];
                wv[i] = mx_i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
            }
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                const mx_u32x4 v = at[(WF + wm * MB + m) * WAVE];
                const mx_i32x8 xv = {(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < NF; ++i) acc[i][m] = mx_mfma4(wv[i], xv, acc[i][m], b, sw[i], sx[m]);
            }
            if constexpr (MULTI) {
                if (--left == 0 || t == last) {
                    const bool first = t < A.CT;
                    left = A.CT;
#pragma unroll
                    for (int i = 0; i < NF; ++i)
#pragma unroll
                        for (int m = 0; m < MB; ++m) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) tot[i][m][e] = first ? acc[i][m][e] : tot[i][m][e] + acc[i][m][e];
                            acc[i][m] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
                        }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            const int64_t r = (x0 + wm * MB + m) * 16 + col, f = f0 + wn * NF + i;
            if (r >= A.M || f >= frags) continue;
            mx_f32x4 o;
            if constexpr (MULTI) o = tot[i][m];
            else o = acc[i][m];
            mx_store(A, r, (int)f * 16 + 4 * q, o);
        }
}

// 16-row tiles of x per workgroup, of the ones there are kernels for: the fewest rounds of 256 workgroups, by their
// length (a tile of W costs about what one of x does)
__host__ inline int mx_rows(int M, int64_t ntiles, std::initializer_list<int> mbs) {
    int best = 0;
    int64_t cost = 0;
    for (const int mb : mbs) {
        const int64_t wgs = (M + 16 * mb - 1) / (16 * mb) * ntiles, c = (wgs + 255) / 256 * (mb + 1);
        if (!best || c < cost) best = mb, cost = c;
    }
    return best;
}

template <int XM, bool DMA, int MB, bool MULTI>
static int mx_launch_tile(const MxArgs& a, hipStream_t st) {
    const int mtiles = (a.M + 16 * MB - 1) / (16 * MB), ntiles = (int)((mx_frags(a.N) + 15) / 16);
    hipLaunchKernelGGL((mx4_tile_kernel<XM, DMA, 4, MB, MULTI>), dim3(mx_grid(mtiles, ntiles)), dim3(256), 2 * 16 * MB * 256, st, a,
                       mtiles, ntiles);
    return DKV_OK;
}
template <int XM, bool DMA>
static int mx_launch_rows(const MxArgs& a, hipStream_t st) {
    const int64_t ntiles = (mx_frags(a.N) + 15) / 16;
    if (a.S > 1)
        switch (mx_rows(a.M, ntiles, {4, 2})) {
            case 4: return mx_launch_tile<XM, DMA, 4, true>(a, st);
            default: return mx_launch_tile<XM, DMA, 2, true>(a, st);
        }
    switch (mx_rows(a.M, ntiles, {8, 5, 4, 2})) {
        case 8: return mx_launch_tile<XM, DMA, 8, false>(a, st);
        case 5: return mx_launch_tile<XM, DMA, 5, false>(a, st);
        case 4: return mx_launch_tile<XM, DMA, 4, false>(a, st);
        default: return mx_launch_tile<XM, DMA, 2, false>(a, st);
    }
}
template <int MB, bool MULTI>
static int mx_launch_tile4(const MxArgs& a, hipStream_t st) {
    const size_t lds = 2 * (16 + 2 * MB) * 1024;
    auto fn = mx4_tile4_kernel<MB, MULTI>;
    const int mtiles = (a.M + 32 * MB - 1) / (32 * MB), ntiles = (int)((mx_frags(a.N) + 15) / 16);
    hipLaunchKernelGGL(fn, dim3(mx_grid(mtiles, ntiles)), dim3(512), lds, st, a, mtiles, ntiles);
    return DKV_OK;
}

}  // namespace dkv

extern "C" int64_t dkv_mx4_code_bytes(int32_t rows, int32_t k) {
    return rows < 1 || k < 1 ? 0 : dkv::mx_frags(rows) * dkv::mx_tiles(k) * 1024;
}

extern "C" int64_t dkv_mx4_scale_bytes(int32_t rows, int32_t k) {
    return rows < 1 || k < 1 ? 0 : dkv::mx_frags(rows) * dkv::mx_quads(k) * 256;
}

extern "C" int dkv_mx4_quantize(const void* x, int32_t x_dtype, int32_t rows, int32_t k, uint8_t* codes, uint8_t* scales, float* values,
                                dkv_stream_t stream) {
    using namespace dkv;
    DKV_REQUIRE(x && codes && scales, "dkv_mx4_quantize: NULL argument");
    DKV_REQUIRE(x_dtype == DKV_F32 || x_dtype == DKV_BF16, "dkv_mx4_quantize: bad input dtype");
    DKV_REQUIRE(rows >= 0 && k > 0, "dkv_mx4_quantize: bad shape");
    DKV_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
                "dkv_mx4_quantize: codes must be 16-byte and scales 4-byte aligned");
    if (rows == 0) return DKV_OK;
    const int64_t wgs = mx_frags(rows) * mx_quads(k);
    DKV_REQUIRE(wgs < (1LL << 31), "dkv_mx4_quantize: too many values");
    if (x_dtype == DKV_F32)
        hipLaunchKernelGGL((mx4_quantize_kernel<float>), dim3((unsigned)wgs), dim3(256), 0, as_stream(stream),
                           static_cast<const float*>(x), rows, k, codes, reinterpret_cast<uint32_t*>(scales), values);
    else
        hipLaunchKernelGGL((mx4_quantize_kernel<uint16_t>), dim3((unsigned)wgs), dim3(256), 0, as_stream(stream),
                           static_cast<const uint16_t*>(x), rows, k, codes, reinterpret_cast<uint32_t*>(scales), values);
    return check_launch("dkv_mx4_quantize");
}

extern "C" int dkv_mx4_values(const uint8_t* codes, const uint8_t* scales, int32_t rows, int32_t k, float* out, dkv_stream_t stream) {
    using namespace dkv;
    DKV_REQUIRE(codes && scales && out, "dkv_mx4_values: NULL argument");
    DKV_REQUIRE(rows >= 0 && k > 0 && ((int64_t)rows * k + 255) / 256 < (1LL << 31), "dkv_mx4_values: bad shape");
    if (rows == 0) return DKV_OK;
    hipLaunchKernelGGL(mx4_values_kernel, dim3((unsigned)(((int64_t)rows * k + 255) / 256)), dim3(256), 0, as_stream(stream), codes,
                       scales, rows, k, out);
    return check_launch("dkv_mx4_values");
}

extern "C" int dkv_gemm_mx4(const void* x, int32_t x_dtype, const uint8_t* x_scales, const uint8_t* w, const uint8_t* w_scales,
                            const void* bias, int32_t bias_dtype, int32_t M, int32_t N, int32_t K, void* y, int32_t y_dtype,
                            int32_t flags, dkv_stream_t stream) {
    using namespace dkv;
    DKV_REQUIRE(x && w && w_scales && y, "dkv_gemm_mx4: NULL argument");
    DKV_REQUIRE(x_dtype == DKV_F32 || x_dtype == DKV_BF16 || x_dtype == DKV_MX4, "dkv_gemm_mx4: bad input dtype");
    DKV_REQUIRE(x_dtype != DKV_MX4 || x_scales, "dkv_gemm_mx4: 4-bit rows need their scales");
    DKV_REQUIRE(y_dtype == DKV_F32 || y_dtype == DKV_BF16, "dkv_gemm_mx4: bad output dtype");
    DKV_REQUIRE(!bias || bias_dtype == DKV_F32 || bias_dtype == DKV_BF16, "dkv_gemm_mx4: bad bias dtype");
    DKV_REQUIRE(M >= 0 && N > 0 && K > 0, "dkv_gemm_mx4: bad shape");
    DKV_REQUIRE((flags & ~DKV_GEMM_SWIGLU) == 0, "dkv_gemm_mx4: unknown flags");
    const bool swiglu = flags & DKV_GEMM_SWIGLU;
    DKV_REQUIRE(!swiglu || (N % 2 == 0 && !bias), "dkv_gemm_mx4: SwiGLU needs an even N and takes no bias");
    auto aligned = [](const void* p, int a) { return reinterpret_cast<uintptr_t>(p) % a == 0; };
    DKV_REQUIRE(aligned(w, 16) && aligned(w_scales, 4) && aligned(x_scales, 4) && (x_dtype != DKV_MX4 || aligned(x, 16)),
                "dkv_gemm_mx4: codes must be 16-byte and scales 4-byte aligned");
    DKV_REQUIRE(aligned(y, 16), "dkv_gemm_mx4: y must be 16-byte aligned");
    if (M == 0) return DKV_OK;
    MxArgs a = {};
    a.x = x, a.xs = reinterpret_cast<const uint32_t*>(x_scales), a.w = w, a.ws = reinterpret_cast<const uint32_t*>(w_scales);
    a.bias = bias, a.bias_f32 = bias_dtype == DKV_F32, a.y_f32 = y_dtype == DKV_F32, a.swiglu = swiglu;
    a.vec = K % 8 == 0 && aligned(x, 16);
    a.M = M, a.N = N, a.K = K, a.tiles = (int)mx_tiles(K), a.quads = (int)mx_quads(K), a.y = y;
    mx_chunks(N, K, a.S, a.CT);
    hipStream_t st = as_stream(stream);
    if (M > 64 && (x_dtype == DKV_MX4 || a.vec)) {
        int rc;
        if (x_dtype == DKV_MX4) {
            const int64_t ntiles = (mx_frags(N) + 15) / 16;
            // (rows of two waves: 32 MB)
            if (a.S > 1) rc = mx_launch_tile4<4, true>(a, st);
            else if (mx_rows((M + 1) / 2, ntiles, {8, 4}) == 8) rc = mx_launch_tile4<8, false>(a, st);
            else rc = mx_launch_tile4<4, false>(a, st);
        } else if (x_dtype == DKV_F32) {
            rc = mx_launch_rows<MX_XF32, false>(a, st);
        } else if (K % 128 == 0 && (int64_t)M * K < (1LL << 31)) {   // (32-bit byte offsets)
            rc = mx_launch_rows<MX_XBF16, true>(a, st);
        } else {
            rc = mx_launch_rows<MX_XBF16, false>(a, st);
        }
        return rc ? rc : check_launch("dkv_gemm_mx4");
    }
    const int mb = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    const dim3 grid((unsigned)mx_frags(N), (unsigned)((M + 16 * mb - 1) / (16 * mb))), blk(64 * a.S);
    DKV_REQUIRE(grid.y <= 65535, "dkv_gemm_mx4: too many rows");
    const size_t lds = a.S > 1 ? (size_t)a.S * mb * 1024 : 0;
#define DKV_MX(XX)                                                                                    \
    do {                                                                                              \
        if (mb == 1) hipLaunchKernelGGL((mx4_gemm_kernel<XX, 1>), grid, blk, lds, st, a);             \
        else if (mb == 2) hipLaunchKernelGGL((mx4_gemm_kernel<XX, 2>), grid, blk, lds, st, a);        \
        else hipLaunchKernelGGL((mx4_gemm_kernel<XX, 4>), grid, blk, lds, st, a);                     \
    } while (0)
    if (x_dtype == DKV_F32) DKV_MX(MX_XF32);
    else if (x_dtype == DKV_BF16) DKV_MX(MX_XBF16);
    else DKV_MX(MX_XMX4);
#undef DKV_MX
    return check_launch("dkv_gemm_mx4");
}
