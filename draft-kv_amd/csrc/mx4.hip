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
// consecutive values of one row. Bound by memory: bf16 28672 x 4096 with the values written as float32 beside the codes
// 155 to 159 us (5.0 TB/s), 70 % of the bytes the values'.
template <class X>
__device__ __forceinline__ float mx_load(const X* p);
template <>
__device__ __forceinline__ float mx_load(const float* p) { return *p; }
template <>
__device__ __forceinline__ float mx_load(const uint16_t* p) { return bf16_to_f32(*p); }

// VEC: rows of x (and of values) in whole, 16-byte aligned runs of 8.
template <class X, bool VEC>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(const X* __restrict__ x, int rows, int K, uint8_t* __restrict__ codes,
                                                           uint32_t* __restrict__ scales, float* __restrict__ values) {
    __shared__ __align__(16) uint32_t sc[16 * 4];   // [q][c] words of four tiles
    const int64_t quads = mx_quads(K), tiles = mx_tiles(K);
    const int64_t f = blockIdx.x / quads, quad = blockIdx.x % quads;
    const int tid = threadIdx.x, sub = tid % 4, b = tid % 64 / 4;   // block b of the 16 of the row's 512 k
    const int64_t k0 = quad * 512 + 32 * b + 8 * sub;
    const int64_t tile = quad * 4 + b / 4;
    const int c0 = tid / 64;   // rows c0, c0 + 4, ..: all loaded before the first is used
    float v[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t r = f * 16 + c0 + 4 * j;
        const X* p = x + r * K + k0;
        if constexpr (VEC) {
            const bool in = r < rows && k0 < K;
            if constexpr (sizeof(X) == 4) {
                const mx_f32x4 z = {0.f, 0.f, 0.f, 0.f};
                const mx_f32x4 lo = in ? reinterpret_cast<const mx_f32x4*>(p)[0] : z, hi = in ? reinterpret_cast<const mx_f32x4*>(p)[1] : z;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = i < 4 ? lo[i] : hi[i - 4];
            } else {
                const mx_u32x4 w = in ? *reinterpret_cast<const mx_u32x4*>(p) : mx_u32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = r < rows && k0 + i < K ? mx_load(p + i) : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = c0 + 4 * j;
        const int64_t r = f * 16 + c;
        uint32_t a = 0;   // magnitudes order as their bits do; NaN and infinity come out largest
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(v[j][i]) & 0x7fffffffu);
        a = max(a, (uint32_t)__shfl_xor((int)a, 1));
        a = max(a, (uint32_t)__shfl_xor((int)a, 2));
        const int ex = a >> 23;
        const uint32_t s = a == 0 ? 127u : ex == 255 ? (uint32_t)MX_NAN : (uint32_t)max(ex - 2, 1);
        const float scale = __uint_as_float(s << 23);
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][0], v[j][1], scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][2], v[j][3], scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][4], v[j][5], scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[j][6], v[j][7], scale, 3);
        if (tile < tiles)
            *reinterpret_cast<uint32_t*>(codes + (f * tiles + tile) * 1024 + (b % 4 * 16 + c) * 16 + 4 * sub) = w;
        if (sub == 0) reinterpret_cast<uint8_t*>(sc)[(b % 4 * 16 + c) * 4 + b / 4] = (uint8_t)s;
        if (values && r < rows && k0 < K) {
            const mx_f32x2 o[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1),
                                   __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3)};
            float* to = values + r * K + k0;
            if constexpr (VEC) {
                __builtin_nontemporal_store((mx_f32x4{o[0][0], o[0][1], o[1][0], o[1][1]}), reinterpret_cast<mx_f32x4*>(to));
                __builtin_nontemporal_store((mx_f32x4{o[2][0], o[2][1], o[3][0], o[3][1]}), reinterpret_cast<mx_f32x4*>(to) + 1);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (k0 + i < K) to[i] = o[i / 2][i % 2];
            }
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
    int bias_f32, y_f32, swiglu;
    int M, N, K, tiles, quads;
    int ldx;                   // row stride of x in values
    int S, CT;                 // chunks, tiles per chunk
    float* part;               // per-chunk sums [S][M][16 ceil(N / 16)] where each workgroup takes one chunk
    void* y;
};

// K chunks of a weight: one where its row fragments alone give a thousand waves, else about two thousand, of four
// tiles or a multiple. (Chunks double the accumulators of the kernels for many rows: none for the wide weights.)
__host__ inline void mx_chunks(int N, int K, int& S, int& CT) {
    const int tiles = (int)mx_tiles(K);
    S = N >= 16384 ? 1 : std::min(8, (32768 + N - 1) / N);
    CT = ((tiles + S - 1) / S + 3) / 4 * 4;   // whole scale words
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

__device__ __forceinline__ float mx_swiglu(float gate, float up) { return gate / (1.0f + __expf(-gate)) * up; }
__device__ __forceinline__ mx_f32x4 mx_bias4(const MxArgs& A, int n) {
    mx_f32x4 b;
#pragma unroll
    for (int e = 0; e < 4; ++e) b[e] = n + e < A.N ? load_elem(A.bias, n + e, A.bias_f32 ? DKV_F32 : DKV_BF16) : 0.0f;
    return b;
}
// outputs (m, n .. n + 3), n a multiple of 4
__device__ __forceinline__ void mx_store(const MxArgs& A, int64_t m, int n, mx_f32x4 t) {
    if (n >= A.N) return;   // the last fragment's rows past N
    if (A.swiglu) {   // rows of W interleave (gate, up); N is even
        for (int e = 0; e < 4; e += 2)
            if (n + e < A.N) {
                const float o = mx_swiglu(t[e], t[e + 1]);
                const int64_t at = m * (A.N / 2) + (n + e) / 2;
                if (A.y_f32) static_cast<float*>(A.y)[at] = o;
                else static_cast<uint16_t*>(A.y)[at] = f32_to_bf16_rne(o);
            }
        return;
    }
    if (A.bias) t += mx_bias4(A, n);
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

// outputs (m, n .. n + 7), n and N multiples of 8
__device__ __forceinline__ void mx_store8(const MxArgs& A, int64_t m, int n, mx_f32x4 a, mx_f32x4 b) {
    if (A.swiglu) {
        const mx_f32x4 o = {mx_swiglu(a[0], a[1]), mx_swiglu(a[2], a[3]), mx_swiglu(b[0], b[1]), mx_swiglu(b[2], b[3])};
        const int64_t at = m * (A.N / 2) + n / 2;
        if (A.y_f32) *reinterpret_cast<mx_f32x4*>(static_cast<float*>(A.y) + at) = o;
        else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(A.y) + at) = make_uint2(mx_bf16_pair(o[0], o[1]), mx_bf16_pair(o[2], o[3]));
        return;
    }
    if (A.bias) a += mx_bias4(A, n), b += mx_bias4(A, n + 4);
    const int64_t at = m * A.N + n;
    if (A.y_f32) {
        *reinterpret_cast<mx_f32x4*>(static_cast<float*>(A.y) + at) = a;
        *reinterpret_cast<mx_f32x4*>(static_cast<float*>(A.y) + at + 4) = b;
    } else {
        *reinterpret_cast<mx_u32x4*>(static_cast<uint16_t*>(A.y) + at) =
            mx_u32x4{mx_bf16_pair(a[0], a[1]), mx_bf16_pair(a[2], a[3]), mx_bf16_pair(b[0], b[1]), mx_bf16_pair(b[2], b[3])};
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

// A chunk's sums into mx_lds, added in order by the waves, and out. acc: fragments f0 .. f0 + NF - 1 of W by MB tiles of x.
template <int NF, int MB>
__device__ __forceinline__ void mx_join(const MxArgs& A, mx_f32x4* lds, const mx_f32x4 (&acc)[NF][MB], int64_t f0, int64_t m0, int chunk,
                                        int S, int lane) {
    const int64_t frags = mx_frags(A.N);
    const int col = lane % 16, q = lane / 16;
    if (S == 1) {
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int j = 0; j < MB; ++j)
                if (m0 + 16 * j + col < A.M && f0 + i < frags) mx_store(A, m0 + 16 * j + col, (int)(f0 + i) * 16 + 4 * q, acc[i][j]);
        return;
    }
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) lds[((chunk * NF + i) * MB + j) * WAVE + lane] = acc[i][j];
    __syncthreads();
    for (int x = chunk; x < NF * MB; x += S) {
        mx_f32x4 t = lds[x * WAVE + lane];
        for (int s = 1; s < S; ++s) t += lds[(s * NF * MB + x) * WAVE + lane];
        const int64_t m = m0 + 16 * (x % MB) + col, f = f0 + x / MB;
        if (m < A.M && f < frags) mx_store(A, m, (int)f * 16 + 4 * q, t);
    }
}

// ---------------------------------------------------------------- product, few rows
// Bound by the stream of W. A wave takes one chunk of NF row fragments of W, in groups of four tiles (one scale word)
// with the next tiles of W and of x (16 MB rows, from L2) in flight as far as registers go: x comes from L2 a
// microsecond late, and a tile's products take a tenth of that. Codes are converted in registers, or go to the 4-bit
// instruction as they are. More fragments per wave halve and quarter the reads of x, which at 64 rows are 16 times a
// fragment's bytes. Grid (group of fragments, group of rows), one wave per chunk; the sums meet in LDS.
// RAG: K is no multiple of 128 (but of 8): x is zero from there on.
// 28672 x 4096 (62 MB, 13.1 us at the rate of a copy): 4-bit rows 11.4 us for one, 13.7 for 32, 17.8 for 64. 4096 x 4096
// (8.9 MB): 5.0 for one, 8.1 for 64; bf16 rows 6.1 for one, 11.7 for 16: each wave converts its W and waits for its x.
template <int XM, int MB, int NF, bool RAG>
__global__ void __launch_bounds__(512) mx4_stream_kernel(MxArgs A) {
#pragma clang fp contract(off)
    extern __shared__ __align__(16) mx_f32x4 mx_lds[];   // [S][NF][MB][64]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int col = lane % 16, q = lane / 16;
    const int64_t f0 = (int64_t)blockIdx.x * NF, m0 = (int64_t)blockIdx.y * 16 * MB, frags = mx_frags(A.N), xfrags = mx_frags(A.M);
    const int t0 = wave * A.CT, t1 = min(t0 + A.CT, A.tiles);
    // bases are wave-uniform, lanes add 32-bit offsets
    const uint8_t* wp[NF];
    const uint32_t* sp[NF];
#pragma unroll
    for (int i = 0; i < NF; ++i) {
        const int64_t f = min(f0 + i, frags - 1);
        wp[i] = A.w + f * A.tiles * 1024;
        sp[i] = A.ws + f * A.quads * 64;
    }
    constexpr int XW = XM == MX_XMX4 ? 1 : XM == MX_XF32 ? 8 : 4;   // 16-byte pieces of a tile per lane and 16 rows
    constexpr int ES = XM == MX_XF32 ? 4 : 2;
    const uint8_t* xp[MB];
    const uint32_t* xsp[MB];
    uint32_t xo[MB];
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        if constexpr (XM == MX_XMX4) {
            const int64_t xf = min(m0 / 16 + j, xfrags - 1);
            xp[j] = static_cast<const uint8_t*>(A.x) + xf * A.tiles * 1024;
            xsp[j] = A.xs + xf * A.quads * 64;
            xo[j] = 16 * lane;
        } else {
            xp[j] = static_cast<const uint8_t*>(A.x) + m0 * A.ldx * ES;
            xo[j] = (uint32_t)((min(m0 + 16 * j + col, (int64_t)A.M - 1) - m0) * A.ldx + 32 * q) * ES;
            xsp[j] = nullptr;
        }
    }
    constexpr int XB = XM == MX_XMX4 || MB * XW <= 8 ? 4 : 1;   // tiles of x in registers
    mx_u32x4 x[XB][MB][XW];
    auto load_x = [&](int b, int t) {
#pragma unroll
        for (int j = 0; j < MB; ++j)
#pragma unroll
            for (int e = 0; e < XW; ++e) {
                if constexpr (XM == MX_XMX4) {
                    x[b][j][e] = *reinterpret_cast<const mx_u32x4*>(xp[j] + (int64_t)t * 1024 + xo[j]);
                } else if constexpr (RAG) {   // (a piece past K: the row's first values, zeroed when used)
                    const bool in = 128 * t + 32 * q + e * (16 / ES) < A.K;
                    x[b][j][e] = *reinterpret_cast<const mx_u32x4*>(xp[j] + (in ? xo[j] + 128 * ES * t + 16 * e : xo[j] - 32 * ES * q));
                } else {
                    x[b][j][e] = *reinterpret_cast<const mx_u32x4*>(xp[j] + (int64_t)t * (128 * ES) + xo[j] + 16 * e);
                }
            }
    };
    auto x_operand = [&](int b, int j, int e, int t) {   // k = 32 q + 8 e .. of the tile, as bf16
        mx_u32x4 v;
        if constexpr (XM == MX_XF32) {
            const mx_u32x4 a = x[b][j][2 * e], c = x[b][j][2 * e + 1];
            v = mx_u32x4{mx_bf16_pair(__uint_as_float(a[0]), __uint_as_float(a[1])), mx_bf16_pair(__uint_as_float(a[2]), __uint_as_float(a[3])),
                         mx_bf16_pair(__uint_as_float(c[0]), __uint_as_float(c[1])), mx_bf16_pair(__uint_as_float(c[2]), __uint_as_float(c[3]))};
        } else {
            v = x[b][j][e];
        }
        if (RAG && 128 * t + 32 * q + 8 * e >= A.K) v = mx_u32x4{0, 0, 0, 0};
        return __builtin_bit_cast(mx_bf16x8, v);
    };
    mx_u32x4 w[4][NF];
    uint32_t sc[NF], sn[NF], xc[MB], xn[MB];   // scale words of the group, and of the next
    auto load_w = [&](int b, int t) {
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            const mx_u32x4* p = reinterpret_cast<const mx_u32x4*>(wp[i] + (int64_t)t * 1024 + 16u * lane);
            w[b][i] = __builtin_nontemporal_load(p);
        }
    };
    auto load_s = [&](int g) {
#pragma unroll
        for (int i = 0; i < NF; ++i) sn[i] = (sp[i] + (int64_t)g * 64)[(uint32_t)lane];
        if constexpr (XM == MX_XMX4) {
#pragma unroll
            for (int j = 0; j < MB; ++j) xn[j] = (xsp[j] + (int64_t)g * 64)[(uint32_t)lane];
        }
    };
    mx_f32x4 acc[NF][MB];
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
    load_s(t0 / 4);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        if (XB == 4) load_x(b, min(t0 + b, t1 - 1));
        load_w(b, min(t0 + b, t1 - 1));
    }
    for (int tb = t0; tb < t1; tb += 4) {
#pragma unroll
        for (int i = 0; i < NF; ++i) sc[i] = sn[i];
        if constexpr (XM == MX_XMX4) {
#pragma unroll
            for (int j = 0; j < MB; ++j) xc[j] = xn[j];
        }
        load_s(min(tb / 4 + 1, (t1 - 1) / 4));
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int t = tb + b, xb = XB == 4 ? b : 0;
            if (t >= t1) break;   // uniform
            if (XB == 1) load_x(0, t);
            if constexpr (XM == MX_XMX4) {
#pragma unroll
                for (int i = 0; i < NF; ++i) {
                    const mx_i32x8 wv = {(int)w[b][i][0], (int)w[b][i][1], (int)w[b][i][2], (int)w[b][i][3], 0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < MB; ++j) {
                        const mx_u32x4 v = x[xb][j][0];
                        acc[i][j] = mx_mfma4(wv, mx_i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0}, acc[i][j], b, sc[i], xc[j]);
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    mx_bf16x8 xv[MB];
#pragma unroll
                    for (int j = 0; j < MB; ++j) xv[j] = x_operand(xb, j, e, t);
#pragma unroll
                    for (int i = 0; i < NF; ++i) {
                        const mx_bf16x8 wv = mx_operand(w[b][i][e], __uint_as_float((sc[i] >> 8 * b & 0xff) << 23));
#pragma unroll
                        for (int j = 0; j < MB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[j], acc[i][j], 0, 0, 0);
                    }
                }
            }
            if (XB == 4) load_x(b, min(t + 4, t1 - 1));
            load_w(b, min(t + 4, t1 - 1));
        }
    }
    mx_join<NF, MB>(A, mx_lds, acc, f0, m0, wave, A.S, lane);
}

// A wave's outputs: fragments f0 .. of W by rows m0 .. of x, o[NF][MB] as the matrix instructions leave them: a lane has
// four outputs of each fragment, 32 bytes of a row where they are bf16. 16 rows at a time pass through LDS (the wave's
// own) and leave in runs of 16 NF. 4096 x 28672 from 4096 in 4 bits: 256 us, with every lane's own stores 321 (a workgroup
// alone on its CU has nothing else to do meanwhile); bf16 rows 657 and 685. Rows of odd length (50257) leave value by value.
template <int NF, int MB>
__device__ __forceinline__ void mx_store_tile(const MxArgs& A, float* lds, const mx_f32x4* o, int64_t f0, int64_t m0, int lane) {
    const int64_t frags = mx_frags(A.N);
    const int col = lane % 16, q = lane / 16;
    if (A.N % 8 == 0) {   // 16 bytes per lane (SwiGLU: half)
        constexpr int W = 16 * NF, LD = W + 4, ROWS = WAVE / (W / 8);
        const int n = lane % (W / 8) * 8, rr = lane / (W / 8);
        const int64_t gn = f0 * 16 + n;
#pragma unroll
        for (int m = 0; m < MB; ++m) {
#pragma unroll
            for (int i = 0; i < NF; ++i) *reinterpret_cast<mx_f32x4*>(lds + col * LD + 16 * i + 4 * q) = o[i * MB + m];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int x = 0; x < 16; x += ROWS) {
                const int64_t r = m0 + 16 * m + x + rr;
                const mx_f32x4* v = reinterpret_cast<const mx_f32x4*>(lds + (x + rr) * LD + n);
                if (r < A.M && gn < A.N) mx_store8(A, r, (int)gn, v[0], v[1]);
            }
            __builtin_amdgcn_wave_barrier();
        }
        return;
    }
    if (A.swiglu) {
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                const int64_t r = m0 + 16 * m + col;
                if (r < A.M && f0 + i < frags) mx_store(A, r, (int)(f0 + i) * 16 + 4 * q, o[i * MB + m]);
            }
        return;
    }
    constexpr int W = 16 * NF, ROWS = WAVE / W;   // outputs of a row, rows per turn
    const int n = lane % W, rr = lane / W;
    const int64_t gn = f0 * 16 + n;
    const float bias = A.bias && gn < A.N ? load_elem(A.bias, gn, A.bias_f32 ? DKV_F32 : DKV_BF16) : 0.0f;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) lds[col * (W + 1) + 16 * i + 4 * q + e] = o[i * MB + m][e];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int x = 0; x < 16; x += ROWS) {
            const int64_t r = m0 + 16 * m + x + rr;
            float v = lds[(x + rr) * (W + 1) + n];
            if (A.bias) v += bias;
            if (r < A.M && gn < A.N) {
                if (A.y_f32) static_cast<float*>(A.y)[r * A.N + gn] = v;
                else static_cast<uint16_t*>(A.y)[r * A.N + gn] = f32_to_bf16_rne(v);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---------------------------------------------------------------- product, many rows
// One workgroup: BN rows of W x BM rows of x, in steps of one tile (128 k). The order of the workgroups gives each XCD
// (workgroup g runs on XCD g % 8) one contiguous run of tiles, up to GM tiles of x by one of W at a time, so the 32 CUs
// of an XCD share both in its L2.
constexpr int MX_GM = 8;
__device__ __forceinline__ bool mx_tile_of(int mtiles, int ntiles, int& mt, int& nt) {
    const int total = mtiles * ntiles, per = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= total) return false;
    const int groups = (mtiles + MX_GM - 1) / MX_GM, gm = (mtiles + groups - 1) / groups;
    const int first = id / (gm * ntiles) * gm, r = id - first * ntiles, n = min(gm, mtiles - first);
    mt = first + r % n, nt = r / n;
    return true;
}
__host__ inline unsigned mx_grid(int mtiles, int ntiles) { return (unsigned)((mtiles * ntiles + 7) / 8 * 8); }

// bf16 rows of whole tiles (others are packed first): four waves, NF fragments of W (16 NF rows) each, against the same
// 16 MB rows of x. W's codes go from memory to registers PD tiles ahead and are converted there (a conversion per two
// values, a ninth of the matrix instructions' time at NF x MB = 4 x 8); x goes straight to LDS, PD + 1 stages. LDS holds
// x by rows of 16 pieces (8 values), piece p of row r in slot p ^ (r % 16): a row's pieces arrive together, and the 16
// rows that an operand read takes lie on different banks. One tile ahead is enough where two workgroups per CU multiply
// a thousand cycles per tile; a few rows' tiles are shorter than W's way from memory.
// 28672 x 4096: one row 15 us, 32 rows 16, 80 rows 27, 160 rows 40 (930 TFLOP/s; without the operands of a step ahead 50), 1100 rows
// 190, 4096 rows 657 (1460 TFLOP/s, what a large bf16 product of the library reaches).
enum { MX_CHAIN, MX_MULTI, MX_PART };   // one chunk; several, added here; one of several, to memory
template <int NF, int MB, int PD, int MODE>
__global__ void __launch_bounds__(256, 2) mx4_tile_kernel(MxArgs A, int mtiles, int ntiles) {
#pragma clang fp contract(off)
    constexpr bool MULTI = MODE == MX_MULTI;
    constexpr int BM = 16 * MB, STAGE = BM * 256, NS = PD + 1;
    static_assert(NS == 2 || NS == 4, "a group of four tiles takes whole turns of the stages");
    extern __shared__ __align__(16) char mx_smem[];   // [NS][BM][16 slots] of 16 bytes
    int mt, nt;
    if (!mx_tile_of(mtiles, ntiles, mt, nt)) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE;
    const int col = lane % 16, q = lane / 16;
    const int64_t m0 = (int64_t)mt * BM;
    const int64_t frags = mx_frags(A.N), f0 = ((int64_t)nt * 4 + wave) * NF;
    const uint8_t* wp[NF];
    const uint32_t* sp[NF];
#pragma unroll
    for (int i = 0; i < NF; ++i) {
        const int64_t f = min(f0 + i, frags - 1);
        wp[i] = A.w + f * A.tiles * 1024;
        sp[i] = A.ws + f * A.quads * 64;
    }
    const int first = MODE == MX_PART ? (int)blockIdx.y * A.CT : 0;
    const int last = MODE == MX_PART ? min(first + A.CT, A.tiles) - 1 : A.tiles - 1;
    uint32_t xoff[MB];   // byte offset of this lane's piece i of tile 0: row 4 (wave + 4 i) + q, slot col
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int r = 4 * (wave + 4 * i) + q;
        xoff[i] = (uint32_t)(2 * (min(m0 + r, (int64_t)A.M - 1) * A.ldx + 8 * (col ^ (r & 15))));
    }
    mx_u32x4 w[NS][NF];
    uint32_t sc[NF], sn[NF];   // scale words of the group, and of the next
    // tile t (b = t % 4) into stage b % NS; past the last it again, so that every step issues the same loads. With a
    // group's first tile come its scales.
    auto fetch = [&](int t, int b) {
        const int tn = min(t, last);
        const uint32_t base = lds_offset(mx_smem) + b % NS * STAGE;
#pragma unroll
        for (int i = 0; i < MB; ++i)
            dma_b128<false>(static_cast<const char*>(A.x) + (int64_t)tn * 256, xoff[i], base + (wave + 4 * i) * 1024);
#pragma unroll
        for (int i = 0; i < NF; ++i) w[b % NS][i] = *reinterpret_cast<const mx_u32x4*>(wp[i] + (int64_t)tn * 1024 + 16u * lane);
        if (b == 0) {
#pragma unroll
            for (int i = 0; i < NF; ++i) sn[i] = (sp[i] + (int64_t)(tn / 4) * 64)[(uint32_t)lane];
        }
    };
    mx_f32x4 acc[NF][MB], tot[MULTI ? NF : 1][MULTI ? MB : 1];
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < PD; ++b) fetch(first + b, b);
    int left = A.CT;
    for (int t0 = first; t0 <= last; t0 += 4) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int t = t0 + b;
            if (t > last) break;   // uniform
            // tile t is there once at most the loads of the PD - 1 tiles after it are in flight (a group's first has its
            // scales' more); every wave is done with the stage that is fetched into next
            if (PD == 1) wait_loads_barrier<0>();
            else if (b >= 2) wait_loads_barrier<(PD - 1) * (MB + NF) + NF>();
            else wait_loads_barrier<(PD - 1) * (MB + NF)>();
            if (b == 0) {
#pragma unroll
                for (int i = 0; i < NF; ++i) sc[i] = sn[i];
            }
            fetch(t + PD, (b + PD) % 4);
            const char* xs = mx_smem + b % NS * STAGE + col * 256;
            // the operands of step j + 1 are under way while step j multiplies, where registers hold both (and few
            // workgroups share a CU)
            constexpr int AHEAD = PD == 3 && NF * MB <= 20 ? 2 : 1;
            mx_bf16x8 wv[AHEAD][NF], xv[AHEAD][MB];
            auto operands = [&](int j) {
#pragma unroll
                for (int m = 0; m < MB; ++m)
                    xv[j % AHEAD][m] = *reinterpret_cast<const mx_bf16x8*>(xs + m * 4096 + ((4 * q + j) ^ col) * 16);
#pragma unroll
                for (int i = 0; i < NF; ++i)
                    wv[j % AHEAD][i] = mx_operand(w[b % NS][i][j], __uint_as_float((sc[i] >> 8 * b & 0xff) << 23));
            };
            if (AHEAD == 2) operands(0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (AHEAD == 1) operands(j);
                else if (j < 3) operands(j + 1);
                if (AHEAD == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int m = 0; m < MB; ++m)
#pragma unroll
                    for (int i = 0; i < NF; ++i)
                        acc[i][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[j % AHEAD][i], xv[j % AHEAD][m], acc[i][m], 0, 0, 0);
                if (AHEAD == 2) __builtin_amdgcn_sched_barrier(0);
            }
        }
        if constexpr (MULTI) {
            left -= 4;
            if (left == 0 || t0 + 4 > last) {   // a chunk ends
                const bool init = t0 < A.CT;
                left = A.CT;
#pragma unroll
                for (int i = 0; i < NF; ++i)
#pragma unroll
                    for (int m = 0; m < MB; ++m) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) tot[i][m][e] = init ? acc[i][m][e] : tot[i][m][e] + acc[i][m][e];
                        acc[i][m] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
                    }
            }
        }
    }
    wait_loads_barrier<0>();   // the repeated loads of the last tile have landed; LDS is free
    if constexpr (MODE == MX_PART) {
        float* part = A.part + (int64_t)blockIdx.y * A.M * frags * 16;
#pragma unroll
        for (int i = 0; i < NF; ++i)
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                const int64_t r = m0 + 16 * m + col;
                if (r < A.M && f0 + i < frags) *reinterpret_cast<mx_f32x4*>(part + (r * frags + f0 + i) * 16 + 4 * q) = acc[i][m];
            }
        return;
    }
    mx_f32x4* o;
    if constexpr (MULTI) o = &tot[0][0];
    else o = &acc[0][0];
    mx_store_tile<NF, MB>(A, reinterpret_cast<float*>(mx_smem) + wave * (16 * (16 * NF + 4)), o, f0, m0, lane);
}

// The chunks' sums in order, and out: four outputs per thread.
__global__ void __launch_bounds__(256) mx4_reduce_kernel(MxArgs A) {
#pragma clang fp contract(off)
    const int64_t quads = mx_frags(A.N) * 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= quads * A.M) return;
    const mx_f32x4* p = reinterpret_cast<const mx_f32x4*>(A.part) + i;
    mx_f32x4 v[8];
#pragma unroll
    for (int c = 0; c < 8; ++c)
        if (c < A.S) v[c] = p[c * quads * A.M];
    mx_f32x4 t = v[0];
#pragma unroll
    for (int c = 1; c < 8; ++c)
        if (c < A.S) t += v[c];
    mx_store(A, i / quads, (int)(i % quads) * 4, t);
}

// Rows of any type and width as bf16 rows of whole tiles, zeros past K. VEC: rows of x in whole, 16-byte aligned runs of
// 8. Bound by the traffic (4096 x 14336 float32, 352 MB: 62 us, value by value 125).
template <class X, bool VEC>
__global__ void __launch_bounds__(256) mx4_pack_kernel(const X* __restrict__ x, int64_t M, int K, int Kp, uint32_t* __restrict__ out) {
    const int64_t n = M * (Kp / 8);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / (Kp / 8);
        const int k = (int)(i % (Kp / 8)) * 8;
        const X* p = x + r * K + k;
        mx_u32x4 o = {0, 0, 0, 0};
        if constexpr (VEC && sizeof(X) == 4) {
            if (k < K) {
                const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
                o = mx_u32x4{mx_bf16_pair(a.x, a.y), mx_bf16_pair(a.z, a.w), mx_bf16_pair(b.x, b.y), mx_bf16_pair(b.z, b.w)};
            }
        } else if constexpr (VEC) {
            if (k < K) o = *reinterpret_cast<const mx_u32x4*>(p);
        } else {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = k + e < K ? mx_load(p + e) : 0.0f;
            o = mx_u32x4{mx_bf16_pair(v[0], v[1]), mx_bf16_pair(v[2], v[3]), mx_bf16_pair(v[4], v[5]), mx_bf16_pair(v[6], v[7])};
        }
        *reinterpret_cast<mx_u32x4*>(out + i * 4) = o;
    }
}

// 4-bit rows: eight waves, four along W by two along x, 4 x MB fragments each. Both operands' tiles go to LDS as they
// are (1 KB, one load instruction each, four stages); the scale words straight to registers, once in four tiles. At
// 4 x 8 a tile of 256 x 256 reads 32 KB per 1024 cycles of matrix instructions, half of what an XCD's L2 gives its CUs.
// 28672 x 4096: 512 rows 42 us (2.8 PFLOP/s), 4096 rows 256 (3.8): without the matrix instructions 219, without the
// loads 204, so neither alone bounds it; a tile's barrier and the stores at the end do the rest.
template <int MB, bool MULTI>
__global__ void __launch_bounds__(512, 2) mx4_tile4_kernel(MxArgs A, int mtiles, int ntiles) {
#pragma clang fp contract(off)
    constexpr int NF = 4, WF = 4 * NF, XF = 2 * MB, STAGE = (WF + XF) * 1024, PER = (WF + XF) / 8, PD = 3;
    static_assert((WF + XF) % 8 == 0, "a stage's loads split evenly over the waves");
    extern __shared__ __align__(16) char mx_smem[];   // [4][W fragments, x fragments][1 KB]
    int mt, nt;
    if (!mx_tile_of(mtiles, ntiles, mt, nt)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int wn = wave % 4, wm = wave / 4;
    const int64_t frags = mx_frags(A.N), xfrags = mx_frags(A.M), f0 = (int64_t)nt * WF, x0 = (int64_t)mt * XF;
    const char* src[PER];   // this wave's fragments of a stage: wave, wave + 8, ...
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int p = wave + 8 * i;
        src[i] = p < WF ? reinterpret_cast<const char*>(A.w) + min(f0 + p, frags - 1) * A.tiles * 1024
                        : static_cast<const char*>(A.x) + min(x0 + (p - WF), xfrags - 1) * A.tiles * 1024;
    }
    const uint32_t *wsp[NF], *xsp[MB];
#pragma unroll
    for (int i = 0; i < NF; ++i) wsp[i] = A.ws + min(f0 + wn * NF + i, frags - 1) * A.quads * 64;
#pragma unroll
    for (int m = 0; m < MB; ++m) xsp[m] = A.xs + min(x0 + wm * MB + m, xfrags - 1) * A.quads * 64;
    const int last = A.tiles - 1;
    uint32_t sw[NF], sx[MB], nw[NF], nx[MB];   // scale words of the group of four tiles, and of the next
    // tile t (b = t % 4) into stage b; past the last it again, so that every step issues the same loads. With a group's
    // first tile come its scales.
    auto fetch = [&](int t, int b) {
        const int tn = min(t, last);
        const uint32_t base = lds_offset(mx_smem) + b * STAGE;
#pragma unroll
        for (int i = 0; i < PER; ++i) dma_b128<false>(src[i] + (int64_t)tn * 1024, 16 * lane, base + (wave + 8 * i) * 1024);
        if (b == 0) {
#pragma unroll
            for (int i = 0; i < NF; ++i) nw[i] = (wsp[i] + (int64_t)(tn / 4) * 64)[(uint32_t)lane];
#pragma unroll
            for (int m = 0; m < MB; ++m) nx[m] = (xsp[m] + (int64_t)(tn / 4) * 64)[(uint32_t)lane];
        }
    };
    mx_f32x4 acc[NF][MB], tot[MULTI ? NF : 1][MULTI ? MB : 1];
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int j = 0; j < MB; ++j) acc[i][j] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < PD; ++b) fetch(b, b);
    int left = A.CT;
    for (int t0 = 0; t0 <= last; t0 += 4) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int t = t0 + b;
            if (t > last) break;   // uniform
            // (as in mx4_tile_kernel: at most the two tiles after it are in flight, one of them with scales)
            if (b >= 2) wait_loads_barrier<(PD - 1) * PER + NF + MB>();
            else wait_loads_barrier<(PD - 1) * PER>();
            if (b == 0) {
#pragma unroll
                for (int i = 0; i < NF; ++i) sw[i] = nw[i];
#pragma unroll
                for (int m = 0; m < MB; ++m) sx[m] = nx[m];
            }
            fetch(t + PD, (b + PD) % 4);
            const mx_u32x4* at = reinterpret_cast<const mx_u32x4*>(mx_smem + b * STAGE) + lane;
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
        }
        if constexpr (MULTI) {
            left -= 4;
            if (left == 0 || t0 + 4 > last) {
                const bool first = t0 < A.CT;
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
    wait_loads_barrier<0>();   // the repeated loads of the last tile have landed; LDS is free
    mx_f32x4* o;
    if constexpr (MULTI) o = &tot[0][0];
    else o = &acc[0][0];
    mx_store_tile<NF, MB>(A, reinterpret_cast<float*>(mx_smem) + wave * (16 * (16 * NF + 4)), o, f0 + wn * NF, (x0 + wm * MB) * 16, lane);
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

template <int NF, int MB, int PD, int MODE>
static int mx_launch_tile(const MxArgs& a, hipStream_t st) {
    const int mtiles = (a.M + 16 * MB - 1) / (16 * MB), ntiles = (int)((mx_frags(a.N) + 4 * NF - 1) / (4 * NF));
    const size_t lds = (size_t)(PD + 1) * 16 * MB * 256;
    auto fn = mx4_tile_kernel<NF, MB, PD, MODE>;
    static size_t done[16] = {};
    if (!reserve_lds(reinterpret_cast<const void*>(fn), lds, done))
        return fail(DKV_ELAUNCH, "dkv_gemm_mx4: cannot reserve " + std::to_string(lds) + " B of LDS");
    hipLaunchKernelGGL(fn, dim3(mx_grid(mtiles, ntiles), MODE == MX_PART ? a.S : 1), dim3(256), lds, st, a, mtiles, ntiles);
    if (MODE != MX_PART) return DKV_OK;
    const int rc = check_launch("dkv_gemm_mx4");
    if (rc) return rc;
    hipLaunchKernelGGL(mx4_reduce_kernel, dim3((unsigned)((mx_frags(a.N) * 4 * a.M + 255) / 256)), dim3(256), 0, st, a);
    return DKV_OK;
}
// Whether the chunks of a narrow W go to workgroups of their own, their sums through memory: where the tiles of 32 rows
// by 128 of W are fewer than the CUs and a workgroup is spared enough steps to pay for the sums and their launch.
// N = 4096, bf16, chunks apart against one after another: K = 4096 11.9 us against 16.3 at 32 rows, 20.5 against 16.5
// at 96; K = 14336 16.9 against 50.2 at 32, 43.0 against 52.0 at 160, 68.5 against 60.3 at 320; N = 960, K = 576 9
// against 7.9.
static bool mx_parts(int M, int N, int K) {
    int S, CT;
    mx_chunks(N, K, S, CT);
    return mx_tiles(K) - CT >= (M <= 32 ? 24 : 64) && (M + 31) / 32 * ((mx_frags(N) + 7) / 8) < 256;
}
static size_t mx_part_bytes(int M, int N, int K) {
    int S, CT;
    mx_chunks(N, K, S, CT);
    return mx_parts(M, N, K) ? (size_t)S * M * mx_frags(N) * 64 : 0;
}
static int mx_launch_rows(const MxArgs& a, hipStream_t st) {
    const int64_t wide = (mx_frags(a.N) + 15) / 16, narrow = (mx_frags(a.N) + 7) / 8;   // tiles of W: 256, 128 rows
    if (a.part) return a.M <= 32 ? mx_launch_tile<2, 2, 3, MX_PART>(a, st) : mx_launch_tile<2, 4, 3, MX_PART>(a, st);
    if (a.S > 1) {
        // (the chunks' sums take registers: four tiles of x at most. N = 4096, 64 x 256 against 32 x 128: 52.6 us against
        // 40.8 at 1024 rows, 65.1 against 70.2 at 2048; K = 14336 167 against 116, 194 against 223)
        if ((a.M + 63) / 64 * wide >= 512) return mx_launch_tile<4, 4, 1, MX_MULTI>(a, st);
        return mx_launch_tile<2, 2, 3, MX_MULTI>(a, st);
    }
    // two workgroups of 128 rows of W per CU where 256-row tiles leave less than that (their waves then wait for LDS and
    // the conversions one after another)
    if ((a.M + 79) / 80 * wide < 512) switch (mx_rows(a.M, narrow, {5, 4, 2})) {
        // Four stages of 80 rows leave LDS for two workgroups per CU, two stages for four, which then cover each other's
        // waits, beginnings and ends. 28672 x 4096: 160 rows (448 workgroups) 41.9 us with four stages, 50.7 with two;
        // 20000 x 4096: 400 rows (785) 70.0 and 65.0; 50257 x 768: 160 rows (786) 31.5 and 24.3.
        case 5: return (a.M + 79) / 80 * narrow <= 512 ? mx_launch_tile<2, 5, 3, MX_CHAIN>(a, st) : mx_launch_tile<2, 5, 1, MX_CHAIN>(a, st);
        case 4: return mx_launch_tile<2, 4, 3, MX_CHAIN>(a, st);
        default: return mx_launch_tile<2, 2, 3, MX_CHAIN>(a, st);
    }
    // (A W of 131072 rows or more comes here with few rows too, in tiles of 64: 131072 x 4096 at one row 75 us, at 60 rows 68;
    // tiles of 32 by 128 of W take 52 and 76. No weight of the models here is as wide.)
    switch (mx_rows(a.M, wide, {8, 5, 4})) {
        case 8: return mx_launch_tile<4, 8, 1, MX_CHAIN>(a, st);
        case 5: return mx_launch_tile<4, 5, 3, MX_CHAIN>(a, st);
        default: return mx_launch_tile<4, 4, 3, MX_CHAIN>(a, st);
    }
}
template <int XM, int MB, int NF, bool RAG>
static int mx_launch_stream(const MxArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((mx_frags(a.N) + NF - 1) / NF), (unsigned)((a.M + 16 * MB - 1) / (16 * MB))), blk(64 * a.S);
    const size_t lds = a.S > 1 ? (size_t)a.S * NF * MB * 1024 : 0;
    auto fn = mx4_stream_kernel<XM, MB, NF, RAG>;
    static size_t done[16] = {};
    if (!reserve_lds(reinterpret_cast<const void*>(fn), lds, done))
        return fail(DKV_ELAUNCH, "dkv_gemm_mx4: cannot reserve " + std::to_string(lds) + " B of LDS");
    hipLaunchKernelGGL(fn, grid, blk, lds, st, a);
    return check_launch("dkv_gemm_mx4");
}
// Float rows that a wave takes beside its W from L2; more go through LDS. Of a weight in one chunk (wide) all do: its
// workgroups fill the CUs, and their x comes in time (28672 x 4096 bf16: one row 14.8 us, by the waves themselves 16.5, 16
// rows 15.5 and 21.5; 50257 x 768: 8.0 and 9.6, 9.1 and 13.7), unless K % 128 asks for another launch first. Of the others
// up to MX_ONE rows, which cost a wave next to nothing, or MX_FEW where the chunks are short (6144 x 4096: 16 rows 9.7,
// through LDS 10.4; 4096 x 14336: 22.1 and 14.8, one row 10.7 and 14.0).
constexpr int MX_ONE = 4, MX_FEW = 16;
static int mx_few(int N, int K) {
    int S, CT;
    mx_chunks(N, K, S, CT);
    if (S == 1 && N >= 16384) return K % 128 ? MX_ONE : 0;
    return mx_tiles(K) - CT >= 64 ? MX_ONE : MX_FEW;
}
// Packed first are: rows that no 16-byte loads can read (value by value 2048 x 515 took 13 us at 4 rows, packed 5.5;
// 4096 x 4097 27 and 9); of those that go through LDS, rows of K % 128 != 0 and float32 ones; float32 rows past MX_ONE,
// or of a W that is long enough for its waves' conversions of the same x to cost more than a launch (4096 x 14336, one
// row: 16.1 us, packed 12.7; 4096 x 4096 8.6 and 8.6).
static bool mx_packs(const void* x, int x_dtype, int M, int N, int K) {
    if (x_dtype == DKV_MX4) return false;
    if (K % 8 || reinterpret_cast<uintptr_t>(x) % 16) return true;
    const int few = mx_few(N, K);
    return x_dtype == DKV_F32 ? M > std::min(few, MX_ONE) || mx_frags(N) * mx_tiles(K) > 8192 : M > few && K % 128;
}
template <int MB, bool MULTI>
static int mx_launch_tile4(const MxArgs& a, hipStream_t st) {
    const size_t lds = 4 * (16 + 2 * MB) * 1024;
    auto fn = mx4_tile4_kernel<MB, MULTI>;
    static size_t done[16] = {};
    if (!reserve_lds(reinterpret_cast<const void*>(fn), lds, done))
        return fail(DKV_ELAUNCH, "dkv_gemm_mx4: cannot reserve " + std::to_string(lds) + " B of LDS");
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
    const bool vec = k % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(values) % 16 == 0;
#define DKV_MXQ(XX, VV)                                                                                                          \
    hipLaunchKernelGGL((mx4_quantize_kernel<XX, VV>), dim3((unsigned)wgs), dim3(256), 0, as_stream(stream), static_cast<const XX*>(x), \
                       rows, k, codes, reinterpret_cast<uint32_t*>(scales), values)
    if (x_dtype == DKV_F32 && vec) DKV_MXQ(float, true);
    else if (x_dtype == DKV_F32) DKV_MXQ(float, false);
    else if (vec) DKV_MXQ(uint16_t, true);
    else DKV_MXQ(uint16_t, false);
#undef DKV_MXQ
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
                            int32_t flags, void* work, size_t work_bytes, dkv_stream_t stream) {
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
    a.M = M, a.N = N, a.K = K, a.ldx = K, a.tiles = (int)mx_tiles(K), a.quads = (int)mx_quads(K), a.y = y;
    mx_chunks(N, K, a.S, a.CT);
    hipStream_t st = as_stream(stream);
    if (x_dtype == DKV_MX4) {
        const int64_t f = mx_frags(N), ntiles = (f + 15) / 16;
        // Few rows, or tiles too few for the CUs: two workgroups of 64 rows by 4 fragments per CU, at most (N = K = 4096:
        // 512 rows 23.0 us against 24.9 through LDS, 640 rows 32.0 against 25.2; N = 14336: 320 rows 40.4 against 25.5;
        // N = 4096, K = 14336: 512 rows 43.8 against 65.7).
        if (M <= 64 || (M + 63) / 64 * ((f + 3) / 4) <= 512) {
            // As many fragments of W per wave as leave a workgroup per CU, up to four; past 64 rows four, since the
            // workgroups of the other rows fill the CUs (N = K = 4096: 32 rows 8.3 us with one, 11.9 with four; 256
            // rows 11.6 with four, 15.1 with two).
            if (M <= 16) return mx_launch_stream<MX_XMX4, 1, 1, false>(a, st);
            if (M <= 32) return f >= 512 ? mx_launch_stream<MX_XMX4, 2, 2, false>(a, st) : mx_launch_stream<MX_XMX4, 2, 1, false>(a, st);
            if (f >= 1024 || M > 64) return mx_launch_stream<MX_XMX4, 4, 4, false>(a, st);
            return f >= 512 ? mx_launch_stream<MX_XMX4, 4, 2, false>(a, st) : mx_launch_stream<MX_XMX4, 4, 1, false>(a, st);
        }
        int rc;
        if (a.S > 1) rc = mx_launch_tile4<4, true>(a, st);
        else if (mx_rows((M + 1) / 2, ntiles, {8, 4}) == 8) rc = mx_launch_tile4<8, false>(a, st);   // (32 MB rows each)
        else rc = mx_launch_tile4<4, false>(a, st);
        return rc ? rc : check_launch("dkv_gemm_mx4");
    }
    const bool packs = mx_packs(x, x_dtype, M, N, K);
    const int few = mx_few(N, K);
    // byte offsets into the rows that a workgroup takes are 32 bits: all of few rows, 256 of many
    DKV_REQUIRE(M <= few ? (int64_t)M * a.tiles * 128 * (packs || x_dtype == DKV_BF16 ? 2 : 4) < (1LL << 32) : a.tiles <= 1 << 16,
                "dkv_gemm_mx4: K too large");
    if (M <= few && !packs) {
        const bool rag = K % 128;
        if (x_dtype == DKV_F32) return rag ? mx_launch_stream<MX_XF32, 1, 1, true>(a, st) : mx_launch_stream<MX_XF32, 1, 1, false>(a, st);
        if (M <= MX_ONE) return rag ? mx_launch_stream<MX_XBF16, 1, 1, true>(a, st) : mx_launch_stream<MX_XBF16, 1, 1, false>(a, st);
        return rag ? mx_launch_stream<MX_XBF16, 1, 2, true>(a, st) : mx_launch_stream<MX_XBF16, 1, 2, false>(a, st);
    }
    int rc = DKV_OK;
    const int kp = 128 * a.tiles;
    const int part = (int)std::min<int64_t>(M, ((1LL << 31) / kp) & ~255LL);   // rows in parts
    if (packs) {
        const size_t need = (size_t)M * kp * 2;
        if (!work || work_bytes < need || !aligned(work, 16))
            return fail(DKV_EWORKSPACE, "dkv_gemm_mx4: workspace too small or not 16-byte aligned (need " + std::to_string(need) + ")");
        const dim3 grid((unsigned)std::min<int64_t>(8192, ((int64_t)M * (kp / 8) + 255) / 256)), blk(256);
        uint32_t* out = static_cast<uint32_t*>(work);
        const bool vec = K % 8 == 0 && aligned(x, 16);
#define DKV_MXP(XX, VV) hipLaunchKernelGGL((mx4_pack_kernel<XX, VV>), grid, blk, 0, st, static_cast<const XX*>(x), (int64_t)M, K, kp, out)
        if (x_dtype == DKV_F32 && vec) DKV_MXP(float, true);
        else if (x_dtype == DKV_F32) DKV_MXP(float, false);
        else if (vec) DKV_MXP(uint16_t, true);
        else DKV_MXP(uint16_t, false);
#undef DKV_MXP
        if ((rc = check_launch("dkv_gemm_mx4(pack)"))) return rc;
        a.x = work, a.ldx = kp;
    }
    if (M <= few) return M <= MX_ONE ? mx_launch_stream<MX_XBF16, 1, 1, false>(a, st) : mx_launch_stream<MX_XBF16, 1, 2, false>(a, st);
    if (mx_parts(M, N, K)) {
        const size_t xb = packs ? (size_t)M * kp * 2 : 0, need = xb + mx_part_bytes(M, N, K);
        if (!work || work_bytes < need || !aligned(work, 16))
            return fail(DKV_EWORKSPACE, "dkv_gemm_mx4: workspace too small or not 16-byte aligned (need " + std::to_string(need) + ")");
        a.part = reinterpret_cast<float*>(static_cast<char*>(work) + xb);
    }
    const int64_t yrow = (int64_t)(swiglu ? N / 2 : N) * (y_dtype == DKV_F32 ? 4 : 2);
    for (int m = 0; m < M && !rc; m += part) {
        MxArgs b = a;
        b.M = std::min(part, M - m);
        b.x = static_cast<const char*>(a.x) + (int64_t)m * a.ldx * 2;
        b.y = static_cast<char*>(y) + m * yrow;
        rc = mx_launch_rows(b, st);
    }
    return rc ? rc : check_launch("dkv_gemm_mx4");
}

extern "C" size_t dkv_gemm_mx4_workspace(const void* x, int32_t x_dtype, int32_t M, int32_t N, int32_t K) {
    using namespace dkv;
    if (M < 1 || N < 1 || K < 1 || x_dtype == DKV_MX4) return 0;
    // (a multiple of 16: the partial sums follow the packed rows)
    return (mx_packs(x, x_dtype, M, N, K) ? (size_t)M * 128 * mx_tiles(K) * 2 : 0) + (M > mx_few(N, K) ? mx_part_bytes(M, N, K) : 0);
}
