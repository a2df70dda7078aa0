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
    const int mb = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    const dim3 grid((unsigned)mx_frags(N), (unsigned)((M + 16 * mb - 1) / (16 * mb))), blk(64 * a.S);
    DKV_REQUIRE(grid.y <= 65535, "dkv_gemm_mx4: too many rows");
    const size_t lds = a.S > 1 ? (size_t)a.S * mb * 1024 : 0;
    hipStream_t st = as_stream(stream);
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
