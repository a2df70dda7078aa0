// Causal attention over the full cache in 8 bits (layout and definition: paged8.h).
// Reference: the read + softmax of draftkv/llama.py:202-218 over the full cache.
//
// For the query row at position p, with lim = p - p % block_size:
//     s_k = q . K_k / sqrt(D), K and V of keys k < lim as code * 2^e, of lim <= k <= p in bf16
//     out = sum_k 2^(s_k - m) V_k / sum_k 2^(s_k - m)        (scores in base 2, m their maximum)
// Two matrix products per 32 keys, both with the keys as the A operand straight from memory (paged8.h's tiles):
//     S^T[16 keys][16 rows] = K . Q^T      (v_mfma_f32_16x16x32_bf16)
//     O^T[16 d][16 rows]   += V^T . P^T
// A code is exact in bf16 and the conversion instruction applies the block's scale, so the products see the values the
// cache stands for. In the S^T accumulator a lane holds keys 4 q + r of two tiles for one row; taking the k-slots of
// the second product in that order, the probabilities never leave their lane. float32 queries and probabilities are
// split into three bf16 parts (NS = 3: 24 bits, as much as float32 has); bf16 queries are whole, and their
// probabilities are rounded once to bf16 (NS = 1), an error of 2^-9 of each, below the output's own rounding.
//
// Order of the sums, the same for every launch: units of 256 keys at absolute positions, each with a softmax of its
// own in steps of 32; a chunk's eight units fold in order; chunks of 2048 keys fold in order; the query's own block
// last. A unit that a row does not see is the empty state, and folding that changes nothing.
#include <algorithm>

#include "paged8.h"
#include "paged_attn.h"

// (every instantiation rounds alike, whatever the compiler would fuse in it)
#pragma clang fp contract(off)

namespace dkv {

typedef __bf16 p8_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 p8_bf16x2 __attribute__((ext_vector_type(2)));
typedef float p8_f32x2 __attribute__((ext_vector_type(2)));
typedef float p8_f32x4 __attribute__((ext_vector_type(4)));

constexpr int P8_UNIT = 256, P8_CHUNK = 2048, P8_UNITS = P8_CHUNK / P8_UNIT;

struct P8Args {
    dkv_paged8_t c;
    int layer, T, Hq;
    bool in_ring;
    int n_chunks;            // chunks that max_len reaches into; slot n_chunks is the rows' own blocks
    int per_slot;            // chunks per workgroup of the walking kernel
    const void* q;
    const int32_t* start;
    const int32_t* count;
    float qscale;            // log2(e) / sqrt(head_dim)
    float* part;             // o [row][n_chunks + 1][DP]
    float2* ml;              // (m, l) [row][n_chunks + 1]
    void* out;
    bool direct;             // the walking kernel covers every key: it writes out itself
};

// The rows of a workgroup's (sequence, KV head): row r is step r / G, query head h G + r % G.
struct P8Rows {
    int s, h, s0, len, T, G, n_rows;
    __device__ __forceinline__ int pos(int r, int bs, int& lim) const {   // the row's position, and its block's start
        const int p = min(s0 + min(r, n_rows - 1) / G, len - 1);
        lim = p & -bs;
        return p;
    }
    __device__ __forceinline__ int64_t row(int r, int Hq) const { return ((int64_t)s * T + r / G) * Hq + h * G + r % G; }
};

__device__ __forceinline__ P8Rows p8_rows(const P8Args& A, int sh) {
    P8Rows R;
    R.h = sh % A.c.n_kv_heads, R.s = sh / A.c.n_kv_heads;
    R.s0 = __builtin_amdgcn_readfirstlane(A.start[R.s]);
    R.T = A.T;
    R.len = R.s0 + __builtin_amdgcn_readfirstlane(p8_new_rows(A.c, A.T, R.s0, A.count, R.s));
    R.G = __builtin_amdgcn_readfirstlane(A.Hq / A.c.n_kv_heads);
    R.n_rows = A.T * R.G;
    return R;
}

// a, b as NS bf16 parts each, into elements k and k + 1
template <int NS>
__device__ __forceinline__ void p8_split(float a, float b, p8_bf16x8 (&o)[NS], int k) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const p8_bf16x2 h = __builtin_convertvector((p8_f32x2){a, b}, p8_bf16x2);
        o[i][k] = h[0], o[i][k + 1] = h[1];
        const uint32_t u = __builtin_bit_cast(uint32_t, h);
        a -= __uint_as_float(u << 16), b -= __uint_as_float(u & 0xffff0000u);
    }
}

__device__ __forceinline__ uint2 p8_words(uint32_t codes, float scale) {   // four codes as bf16
    return make_uint2(
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true)));
}
__device__ __forceinline__ p8_bf16x8 p8_operand(uint2 a, uint2 b) {
    return __builtin_bit_cast(p8_bf16x8, make_uint4(a.x, a.y, b.x, b.y));
}

// Two tiles (32 keys) as a lane holds them: codes, or bf16 rows.
template <int DP>
struct P8Codes {
    static constexpr int PW = DP < 64 ? DP : 64, PB = PW / 4, NP = DP / PW, NW = PB / 4;
    uint32_t k[2][NP][NW], v[2][NP][NW];
    float sk[2], sv[2];
    __device__ __forceinline__ void load(int a, const uint8_t* tile, uint32_t scales, int lane) {
        load_half(k[a], tile, lane);
        load_half(v[a], tile + 16 * DP, lane);
        sk[a] = p8_scale(scales & 0xff), sv[a] = p8_scale(scales >> 8 & 0xff);
    }
    __device__ __forceinline__ static void load_half(uint32_t (&o)[NP][NW], const uint8_t* p, int lane) {
        typedef uint32_t vec __attribute__((ext_vector_type(NW)));
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const vec w = *reinterpret_cast<const vec*>(p + i * 16 * PW + lane * PB);
#pragma unroll
            for (int j = 0; j < NW; ++j) o[i][j] = w[j];
        }
    }
    // A operand of k-step st of tile a
    __device__ __forceinline__ p8_bf16x8 kop(int a, int st) const {
        const int i = st * 32 / PW, w = st * 32 % PW / 16;
        return p8_operand(p8_words(k[a][i][w], sk[a]), p8_words(k[a][i][w + 1], sk[a]));
    }
    // A operand of d-tile dt: keys 4 q .. of tile 0 (if T0), of tile 1 (if T1), else zeros
    __device__ __forceinline__ p8_bf16x8 vop(int dt, bool t0, bool t1) const {
        const int i = dt * 16 / PW, w = dt * 16 % PW / 16;
        const uint2 z = make_uint2(0, 0);
        return p8_operand(t0 ? p8_words(v[0][i][w], sv[0]) : z, t1 ? p8_words(v[1][i][w], sv[1]) : z);
    }
};

template <int DP>
struct P8Bf16 {
    static constexpr int PW = DP < 64 ? DP : 64, PB = PW / 4, NP = DP / PW, NW = PB / 2;
    uint32_t k[2][NP][NW], v[2][NP][NW];
    __device__ __forceinline__ void load(int a, const uint16_t* tile, int lane) {
        load_half(k[a], tile, lane);
        load_half(v[a], tile + 16 * DP, lane);
    }
    __device__ __forceinline__ static void load_half(uint32_t (&o)[NP][NW], const uint16_t* p, int lane) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int j = 0; j < NW; j += 4) {
                const uint4 w = *reinterpret_cast<const uint4*>(p + i * 16 * PW + lane * PB + 2 * j);
                o[i][j] = w.x, o[i][j + 1] = w.y, o[i][j + 2] = w.z, o[i][j + 3] = w.w;
            }
    }
    __device__ __forceinline__ p8_bf16x8 kop(int a, int st) const {
        const int i = st * 32 / PW, w = st * 32 % PW / 8;
        return p8_operand(make_uint2(k[a][i][w], k[a][i][w + 1]), make_uint2(k[a][i][w + 2], k[a][i][w + 3]));
    }
    __device__ __forceinline__ p8_bf16x8 vop(int dt, bool t0, bool t1) const {
        const int i = dt * 16 / PW, w = dt * 16 % PW / 8;
        const uint2 z = make_uint2(0, 0);
        return p8_operand(t0 ? make_uint2(v[0][i][w], v[0][i][w + 1]) : z, t1 ? make_uint2(v[1][i][w], v[1][i][w + 1]) : z);
    }
};

// NQ q-tiles of 16 rows (row r0 + 16 i + lane % 16) and their softmax state.
template <int DP, int NQ, int NS>
struct P8State {
    static constexpr int NSTEP = DP / 32, NDT = DP / 16;
    p8_bf16x8 q[NQ][NSTEP][NS];
    p8_f32x4 acc[NQ][NDT];
    float m[NQ], l[NQ];      // l: the lane's own keys
    int lim[NQ], last[NQ];   // the row's block start, its position

    __device__ __forceinline__ void load_rows(const P8Args& A, const P8Rows& R, int r0, int lane) {
        constexpr int PW = DP < 64 ? DP : 64, PB = PW / 4;
        const int D = A.c.head_dim, col = lane % 16, g = lane / 16;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int r = min(r0 + 16 * i + col, R.n_rows - 1);
            last[i] = R.pos(r, A.c.block_size, lim[i]);
            const int64_t at = R.row(r, A.Hq) * D;
#pragma unroll
            for (int st = 0; st < NSTEP; ++st) {
                const int d0 = st * 32 / PW * PW + g * PB + st * 32 % PW / 32 * 8;
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    x[e] = d0 + e >= D ? 0.0f : NS == 1 ? bf16_to_f32(static_cast<const uint16_t*>(A.q)[at + d0 + e])
                                                        : static_cast<const float*>(A.q)[at + d0 + e] * A.qscale;
#pragma unroll
                for (int e = 0; e < 8; e += 2) p8_split<NS>(x[e], x[e + 1], q[i][st], e);
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) acc[i][dt] = p8_f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void end_unit() {
#pragma unroll
        for (int i = 0; i < NQ; ++i) l[i] = lanegroup_sum(l[i]);
    }

    // scores of the 32 keys of x
    template <class Keys>
    __device__ __forceinline__ void scores(const Keys& x, float (&p)[NQ][8], float qscale) {
        p8_f32x4 s[NQ][2];
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) s[i][a] = p8_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < NSTEP; ++st) {
                const p8_bf16x8 kv = x.kop(a, st);
#pragma unroll
                for (int i = 0; i < NQ; ++i)
#pragma unroll
                    for (int j = 0; j < NS; ++j) s[i][a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv, q[i][st][j], s[i][a], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) p[i][k] = NS == 1 ? s[i][k / 4][k % 4] * qscale : s[i][k / 4][k % 4];
    }
    // scores to probabilities against the running maximum; the sums so far are rescaled
    __device__ __forceinline__ void softmax(float (&p)[NQ][8], p8_bf16x8 (&ph)[NQ][NS]) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            float mx = p[i][0];
#pragma unroll
            for (int k = 1; k < 8; ++k) mx = fmaxf(mx, p[i][k]);
            const float mn = fmaxf(m[i], lanegroup_max(mx));
            const float ms = mn == -INFINITY ? 0.0f : mn;   // a row that sees no key yet: p = 0
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                p[i][k] = exp2_hw(p[i][k] - ms);
                sum += p[i][k];
            }
            const float a = mn == m[i] ? 1.0f : exp2_hw(m[i] - mn);
            l[i] = l[i] * a + sum;
            m[i] = mn;
            if (__any(a != 1.0f)) {
#pragma unroll
                for (int dt = 0; dt < NDT; ++dt) acc[i][dt] *= a;
            }
#pragma unroll
            for (int k = 0; k < 8; k += 2) p8_split<NS>(p[i][k], p[i][k + 1], ph[i], k);
        }
    }
    // every row sees all of x
    template <class Keys>
    __device__ __forceinline__ void step(const Keys& x, float qscale) {
        float p[NQ][8];
        p8_bf16x8 ph[NQ][NS];
        scores(x, p, qscale);
        softmax(p, ph);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            const p8_bf16x8 vv = x.vop(dt, true, true);
#pragma unroll
            for (int i = 0; i < NQ; ++i)
#pragma unroll
                for (int j = 0; j < NS; ++j) acc[i][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, ph[i][j], acc[i][dt], 0, 0, 0);
        }
    }
    // Some rows do not see the tiles at kb, kb + 16 (all of a tile or none, keys below lim): a row takes the sums of
    // the tiles that it sees, so that whatever the others hold (0 * NaN is NaN) stays out of them. One that sees both
    // gets step()'s bits.
    __device__ __forceinline__ void step_tiles(const P8Codes<DP>& x, int kb, float qscale) {
        float p[NQ][8];
        p8_bf16x8 ph[NQ][NS];
        scores(x, p, qscale);
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (kb + k / 4 * 16 >= lim[i]) p[i][k] = -INFINITY;
        softmax(p, ph);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            const p8_bf16x8 both = x.vop(dt, true, true), first = x.vop(dt, true, false);
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                p8_f32x4 t = acc[i][dt], u = acc[i][dt];
#pragma unroll
                for (int j = 0; j < NS; ++j) {
                    t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(both, ph[i][j], t, 0, 0, 0);
                    u = __builtin_amdgcn_mfma_f32_16x16x32_bf16(first, ph[i][j], u, 0, 0, 0);
                }
                acc[i][dt] = kb + 16 < lim[i] ? t : kb < lim[i] ? u : acc[i][dt];
            }
        }
    }
    // The rows' own blocks: keys lim <= k <= last. past: the first position that holds no row (stale memory from there).
    __device__ __forceinline__ void step_own(P8Bf16<DP>& x, int kb, int past, float qscale, int lane) {
        constexpr int NW = P8Bf16<DP>::NW, NP = P8Bf16<DP>::NP;
        const int g = lane / 16;
        float p[NQ][8];
        p8_bf16x8 ph[NQ][NS];
        scores(x, p, qscale);
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int key = kb + k / 4 * 16 + 4 * g + k % 4;
                if (key < lim[i] || key > last[i]) p[i][k] = -INFINITY;
            }
        softmax(p, ph);
        // V: two keys per word
        bool odd = false;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    uint32_t& u = x.v[a][i][w];
                    const int key = kb + 16 * a + 4 * g + 2 * (w % 2);
                    if (key >= past) u = 0;
                    else if (key + 1 >= past) u &= 0xffff;
                    odd = odd || (u & 0x7f80) == 0x7f80 || (u >> 16 & 0x7f80) == 0x7f80;
                }
        if (!__any(odd)) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                const p8_bf16x8 vv = x.vop(dt, true, true);
#pragma unroll
                for (int i = 0; i < NQ; ++i)
#pragma unroll
                    for (int j = 0; j < NS; ++j) acc[i][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, ph[i][j], acc[i][dt], 0, 0, 0);
            }
            return;
        }
        // A NaN or an infinity among them: the sums without them, then each of them into the rows that see its key.
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            const uint4 raw = __builtin_bit_cast(uint4, x.vop(dt, true, true));
            auto odd_halves = [](uint32_t u) {
                return ((u & 0x7f80) == 0x7f80 ? 0xffffu : 0u) | ((u >> 16 & 0x7f80) == 0x7f80 ? 0xffff0000u : 0u);
            };
            const uint4 bad = make_uint4(odd_halves(raw.x), odd_halves(raw.y), odd_halves(raw.z), odd_halves(raw.w));
            const p8_bf16x8 fine = __builtin_bit_cast(p8_bf16x8, make_uint4(raw.x & ~bad.x, raw.y & ~bad.y, raw.z & ~bad.z, raw.w & ~bad.w));
#pragma unroll
            for (int i = 0; i < NQ; ++i)
#pragma unroll
                for (int j = 0; j < NS; ++j) acc[i][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fine, ph[i][j], acc[i][dt], 0, 0, 0);
#pragma nounroll
            for (int kk = 0; kk < 32; ++kk) {
                const int key = kb + kk;
                const uint32_t keep = kk % 16 / 4 == g ? kk % 2 ? 0xffff0000u : 0xffffu : 0u;
                const uint32_t k0 = kk % 4 < 2 ? keep : 0u, k1 = kk % 4 < 2 ? 0u : keep;
                const uint32_t t0 = kk < 16 ? ~0u : 0u;
                const p8_bf16x8 one = __builtin_bit_cast(p8_bf16x8, make_uint4(raw.x & bad.x & k0 & t0, raw.y & bad.y & k1 & t0,
                                                                               raw.z & bad.z & k0 & ~t0, raw.w & bad.w & k1 & ~t0));
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    // (the probability's first part alone: the others' signs would make NaN of an infinity)
                    const p8_f32x4 t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(one, ph[i][0], acc[i][dt], 0, 0, 0);
                    if (key >= lim[i] && key <= last[i]) acc[i][dt] = t;
                }
            }
        }
    }

    // The sealed keys [k0, k1), k0 a unit's start, k1 at most its end. all: a bound that every row's lim reaches
    // (keys below it are seen by all).
    __device__ __forceinline__ void unit(const P8Args& A, const P8Rows& R, int k0, int k1, int all, int lane) {
        const dkv_paged8_t& c = A.c;
        const int bs = c.block_size;
        // tile lane % 16 of the unit: its block and scales (tiles past the end repeat the last)
        const int mine = min(k0 + 16 * (lane % 16), k1 - 1) & -16;
        const uint8_t* blk = p8_block(c, R.s, A.layer, mine);
        const uint8_t* tile = blk + p8_tile_off(c, R.h, mine & (bs - 1));
        const uint32_t sc = *reinterpret_cast<const uint16_t*>(blk + p8_scale_off(c, R.h));
        const uint64_t addr = reinterpret_cast<uint64_t>(tile);
        auto fetch = [&](P8Codes<DP>& x, int step) {
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const int t = 2 * step + a;
                const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)addr, t);
                const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(addr >> 32), t);
                x.load(a, reinterpret_cast<const uint8_t*>(hi << 32 | lo), __builtin_amdgcn_readlane((int)sc, t), lane);
            }
        };
        const int steps = (k1 - k0 + 31) / 32;
        P8Codes<DP> cur, nxt;
        fetch(cur, 0);
#pragma unroll 2
        for (int j = 0; j < steps; ++j) {
            fetch(nxt, min(j + 1, steps - 1));
            const int kb = k0 + 32 * j;
            if (kb + 32 <= all) step(cur, A.qscale);
            else step_tiles(cur, kb, A.qscale);
            cur = nxt;
        }
        end_unit();
    }
    // The rows' own blocks, from the first one's start lo to the last row's position hi
    __device__ __forceinline__ void own_blocks(const P8Args& A, const P8Rows& R, int lo, int hi, int lane) {
        const dkv_paged8_t& c = A.c;
        const int base = R.s0 / c.block_size * c.block_size;
        // (steps at absolute multiples of 32, as a key's place in a step takes part in its rounding)
        for (int kb = lo & -32; kb <= hi; kb += 32) {
            P8Bf16<DP> x;
#pragma unroll
            for (int a = 0; a < 2; ++a) {
                const int pos = min(max(kb + 16 * a, lo), hi & -16);
                x.load(a, A.in_ring ? p8_ring_tile(c, R.s, A.layer, R.h, pos) : p8_hot_tile(c, R.s, R.h, pos, base), lane);
            }
            step_own(x, kb, R.len, A.qscale, lane);
        }
        end_unit();
    }
};

// a row's four channels from d0 of its result; l of the row
template <int NS>
__device__ __forceinline__ void p8_store_out(const P8Args& A, int64_t row, int d0, p8_f32x4 o, float l) {
    const int D = A.c.head_dim;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (d0 + e < D) {
            if constexpr (NS == 1) static_cast<uint16_t*>(A.out)[row * D + d0 + e] = f32_to_bf16_rne(o[e] / l);
            else static_cast<float*>(A.out)[row * D + d0 + e] = o[e] / l;
        }
}

// A sequence without new rows has no query.
template <int NS>
__device__ __forceinline__ void p8_zero_rows(const P8Args& A, const P8Rows& R, int r0, int r1, int tid, int threads) {
    const int D = A.c.head_dim;
    for (int i = tid; i < (min(r1, R.n_rows) - r0) * D; i += threads) {
        const int64_t o = R.row(r0 + i / D, A.Hq) * D + i % D;
        if constexpr (NS == 1) static_cast<uint16_t*>(A.out)[o] = 0;
        else static_cast<float*>(A.out)[o] = 0.0f;
    }
}

// ---------------------------------------------------------------- few rows: one chunk per workgroup
// Grid (KV head x sequence, q-group, chunk or own blocks). Eight waves, one unit of the chunk each, straight from
// memory to registers; their states meet in LDS and leave as the chunk's.
template <int DP, int NQ, int NS>
__global__ void __launch_bounds__(512) paged8_chunk_kernel(P8Args A) {
    constexpr int NDT = DP / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const P8Rows R = p8_rows(A, blockIdx.x);
    const int r0 = blockIdx.y * 16 * NQ, chunk = blockIdx.z, bs = A.c.block_size;
    if (R.len <= R.s0) {
        if (chunk == 0) p8_zero_rows<NS>(A, R, r0, r0 + 16 * NQ, threadIdx.x, 512);
        return;
    }
    int lim0, lim1;
    R.pos(r0, bs, lim0);                                               // the least and the largest of the rows'
    const int last1 = R.pos(min(r0 + 16 * NQ, R.n_rows) - 1, bs, lim1);
    const bool own = chunk == A.n_chunks;
    const int c0 = chunk * P8_CHUNK;
    if (!own && c0 >= lim1) return;
    extern __shared__ __align__(16) char p8_lds[];
    p8_f32x4* so = reinterpret_cast<p8_f32x4*>(p8_lds);                // [units][NDT][64]
    float2* sml = reinterpret_cast<float2*>(p8_lds + P8_UNITS * NDT * 1024);   // [NQ][units][16]
    const int units = own ? 1 : min(P8_UNITS, (lim1 - c0 + P8_UNIT - 1) / P8_UNIT);
    P8State<DP, NQ, NS> st;
    if (wave < units) {
        st.load_rows(A, R, r0, lane);
        st.clear();
        if (own) st.own_blocks(A, R, lim0, last1, lane);
        else {
            const int k0 = c0 + wave * P8_UNIT;
            st.unit(A, R, k0, min(k0 + P8_UNIT, lim1), lim0, lane);
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i)
            if (lane < 16) sml[(i * P8_UNITS + wave) * 16 + lane] = make_float2(st.m[i], st.l[i]);
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        if (i > 0) __syncthreads();
        if (wave < units) {
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) so[(wave * NDT + dt) * WAVE + lane] = st.acc[i][dt];
        }
        __syncthreads();
        for (int x = threadIdx.x; x < NDT * WAVE; x += 512) {   // d-tile x / 64, lane x % 64 of the accumulator
            const int ln = x % WAVE, col = ln % 16, r = r0 + 16 * i + col;
            if (r >= R.n_rows) continue;
            float m = -INFINITY, l = 0.0f;
            p8_f32x4 o = {0.f, 0.f, 0.f, 0.f};
            for (int u = 0; u < units; ++u) {
                const float2 ml = sml[(i * P8_UNITS + u) * 16 + col];
                const p8_f32x4 ou = so[u * NDT * WAVE + x];
                float a, b;
                m = fold_max(m, ml.x, a, b);
                l = fold_sum(l, a, ml.y, b);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fold_sum(o[e], a, ou[e], b);
            }
            const int64_t slot = R.row(r, A.Hq) * (A.n_chunks + 1) + chunk;
            *reinterpret_cast<p8_f32x4*>(A.part + slot * DP + x / WAVE * 16 + ln / 16 * 4) = o;
            if (x < 16) A.ml[slot] = make_float2(m, l);
        }
    }
}

// ---------------------------------------------------------------- many rows: a wave walks its rows' keys
// Grid (KV head x sequence, q-group, slot). Four waves with NQ q-tiles each walk the same chunks; the rows' state over
// the chunks so far lies in LDS.
template <int DP, int NQ, int NS>
__global__ void __launch_bounds__(256) paged8_walk_kernel(P8Args A) {
    constexpr int NDT = DP / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const P8Rows R = p8_rows(A, blockIdx.x);
    const int qg = gridDim.y - 1 - blockIdx.y;   // the last rows see the most keys and go first
    const int r0 = (qg * 4 + wave) * 16 * NQ, bs = A.c.block_size;
    if (r0 >= R.n_rows) return;   // (waves never meet at a barrier)
    if (R.len <= R.s0) {
        if (blockIdx.z == 0) p8_zero_rows<NS>(A, R, r0, r0 + 16 * NQ, lane, WAVE);
        return;
    }
    int lim0, lim1;
    R.pos(r0, bs, lim0);
    const int last1 = R.pos(min(r0 + 16 * NQ, R.n_rows) - 1, bs, lim1);
    const bool own = A.direct || blockIdx.z == gridDim.z - 1;   // this workgroup takes the rows' own blocks
    const int ch0 = A.direct ? 0 : blockIdx.z * A.per_slot;
    const int ch1 = A.direct ? A.n_chunks : own ? ch0 : min(ch0 + A.per_slot, A.n_chunks);
    if (!own && ch0 * P8_CHUNK >= lim1) return;
    extern __shared__ __align__(16) char p8_lds[];
    p8_f32x4* so = reinterpret_cast<p8_f32x4*>(p8_lds) + (int64_t)wave * 2 * NQ * NDT * WAVE + lane;   // chunk, then total
    P8State<DP, NQ, NS> st;
    st.load_rows(A, R, r0, lane);
    float m[2][NQ], l[2][NQ];
    auto wipe = [&](int w) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            m[w][i] = -INFINITY, l[w][i] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) so[((w * NQ + i) * NDT + dt) * WAVE] = p8_f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    // the state in st folded into state w; st becomes the sum
    auto fold = [&](int w) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            float a, b;
            m[w][i] = fold_max(m[w][i], st.m[i], a, b);
            l[w][i] = fold_sum(l[w][i], a, st.l[i], b);
            st.m[i] = m[w][i], st.l[i] = l[w][i];
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                p8_f32x4 o = so[((w * NQ + i) * NDT + dt) * WAVE];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = fold_sum(o[e], a, st.acc[i][dt][e], b);
                so[((w * NQ + i) * NDT + dt) * WAVE] = o;
                st.acc[i][dt] = o;
            }
        }
    };
    auto store_part = [&](int slot) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int r = r0 + 16 * i + lane % 16;
            if (r >= R.n_rows) continue;
            const int64_t ps = R.row(r, A.Hq) * (A.n_chunks + 1) + slot;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
                *reinterpret_cast<p8_f32x4*>(A.part + ps * DP + dt * 16 + lane / 16 * 4) = st.acc[i][dt];
            if (lane < 16) A.ml[ps] = make_float2(st.m[i], st.l[i]);
        }
    };
    if (A.direct) wipe(1);
    for (int ch = ch0; ch < ch1 && ch * P8_CHUNK < lim1; ++ch) {
        wipe(0);
        const int cend = min((ch + 1) * P8_CHUNK, lim1);
        for (int k0 = ch * P8_CHUNK; k0 < cend; k0 += P8_UNIT) {
            st.clear();
            st.unit(A, R, k0, min(k0 + P8_UNIT, cend), lim0, lane);
            fold(0);
        }
        if (A.direct) fold(1);
        else store_part(ch);
    }
    if (!own) return;
    st.clear();
    st.own_blocks(A, R, lim0, last1, lane);
    if (!A.direct) return store_part(A.n_chunks);
    fold(1);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const int r = r0 + 16 * i + lane % 16;
        if (r >= R.n_rows) continue;
        const int64_t row = R.row(r, A.Hq);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) p8_store_out<NS>(A, row, dt * 16 + lane / 16 * 4, st.acc[i][dt], st.l[i]);
    }
}

// ---------------------------------------------------------------- merge
// One wave per row: its chunks in order, its own block last.
template <int NS>
__global__ void __launch_bounds__(256) paged8_merge_kernel(P8Args A, int DP) {
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
    if (row >= (int64_t)A.c.batch * A.T * A.Hq) return;
    const int lane = threadIdx.x % WAVE, D = A.c.head_dim;
    const int s = (int)(row / A.Hq / A.T), t = (int)(row / A.Hq % A.T), s0 = A.start[s];
    const int len = s0 + p8_new_rows(A.c, A.T, s0, A.count, s), p = min(s0 + t, len - 1);
    if (len <= s0) return;   // no new rows: written
    const int lim = p / A.c.block_size * A.c.block_size;
    const int n = min((lim + P8_CHUNK - 1) / P8_CHUNK, A.n_chunks);
    const float* po = A.part + row * (A.n_chunks + 1) * DP;
    const float2* pm = A.ml + row * (A.n_chunks + 1);
    float m = -INFINITY, l = 0.0f, o[P8_MAXD / WAVE] = {};
    auto fold = [&](int slot) {
        const float2 ml = pm[slot];
        float a, b;
        m = fold_max(m, ml.x, a, b);
        l = fold_sum(l, a, ml.y, b);
#pragma unroll
        for (int i = 0; i < P8_MAXD / WAVE; ++i) {
            const int d = lane + WAVE * i;
            if (d < D) o[i] = fold_sum(o[i], a, po[(int64_t)slot * DP + d], b);
        }
    };
    for (int c = 0; c < n; ++c) fold(c);
    fold(A.n_chunks);
#pragma unroll
    for (int i = 0; i < P8_MAXD / WAVE; ++i) {
        const int d = lane + WAVE * i;
        if (d >= D) continue;
        if constexpr (NS == 1) static_cast<uint16_t*>(A.out)[row * D + d] = f32_to_bf16_rne(o[i] / l);
        else static_cast<float*>(A.out)[row * D + d] = o[i] / l;
    }
}

// ---------------------------------------------------------------- plan and launch
struct P8Plan {
    int nq, n_chunks, slots, per_slot;
    bool walk, direct;
    size_t bytes;
};

static P8Plan p8_plan(const dkv_paged8_t& c, int T, int Hq, int max_len) {
    P8Plan p = {};
    const int64_t rows = (int64_t)T * (Hq / c.n_kv_heads), tiles = (rows + 15) / 16;
    p.n_chunks = (max_len + P8_CHUNK - 1) / P8_CHUNK;
    const bool wide = p8_dp(c.head_dim) > 128;
    p.nq = tiles > 1 && !wide ? 2 : 1;
    p.walk = tiles > p.nq;
    p.slots = 1, p.per_slot = p.n_chunks, p.direct = p.walk;
    if (p.walk) {
        const int64_t wgs = (tiles + 4 * p.nq - 1) / (4 * p.nq) * c.n_kv_heads * c.batch;
        // too few workgroups for 256 CUs: the chunks go to several, and their states through memory
        if (wgs < 256 && p.n_chunks > 1) {
            p.direct = false;
            p.slots = (int)std::min<int64_t>(p.n_chunks, (512 + wgs - 1) / wgs);
            p.per_slot = (p.n_chunks + p.slots - 1) / p.slots;
            p.slots = (p.n_chunks + p.per_slot - 1) / p.per_slot;
        }
    }
    if (!p.direct) p.bytes = (size_t)c.batch * T * Hq * (p.n_chunks + 1) * (p8_dp(c.head_dim) + 2) * sizeof(float);
    return p;
}

template <int DP, int NQ, int NS>
static int p8_launch(P8Args& a, const P8Plan& p, hipStream_t st) {
    constexpr int NDT = DP / 16;
    const int64_t tiles = ((int64_t)a.T * (a.Hq / a.c.n_kv_heads) + 15) / 16;
    const int pairs = a.c.n_kv_heads * a.c.batch;
    static size_t done[2][16] = {};
    if (p.walk) {
        const size_t lds = (size_t)4 * 2 * NQ * NDT * 1024;
        const int64_t groups = (tiles + 4 * NQ - 1) / (4 * NQ);
        DKV_REQUIRE(groups <= 65535, "dkv_paged8_attention: too many rows");
        auto fn = paged8_walk_kernel<DP, NQ, NS>;
        if (!reserve_lds(reinterpret_cast<const void*>(fn), lds, done[0]))
            return fail(DKV_ELAUNCH, "dkv_paged8_attention: cannot reserve " + std::to_string(lds) + " B of LDS");
        hipLaunchKernelGGL(fn, dim3(pairs, (int)groups, p.direct ? 1 : p.slots + 1), dim3(256), lds, st, a);
    } else {
        const size_t lds = (size_t)P8_UNITS * NDT * 1024 + NQ * P8_UNITS * 16 * sizeof(float2);
        auto fn = paged8_chunk_kernel<DP, NQ, NS>;
        if (!reserve_lds(reinterpret_cast<const void*>(fn), lds, done[1]))
            return fail(DKV_ELAUNCH, "dkv_paged8_attention: cannot reserve " + std::to_string(lds) + " B of LDS");
        hipLaunchKernelGGL(fn, dim3(pairs, (int)((tiles + NQ - 1) / NQ), p.n_chunks + 1), dim3(512), lds, st, a);
    }
    int rc = check_launch("dkv_paged8_attention");
    if (rc || p.direct) return rc;
    const int64_t rows = (int64_t)a.c.batch * a.T * a.Hq;
    hipLaunchKernelGGL(paged8_merge_kernel<NS>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, DP);
    return check_launch("dkv_paged8_attention(merge)");
}

template <int NS>
static int p8_launch_ns(P8Args& a, const P8Plan& p, hipStream_t st) {
    switch (p8_dp(a.c.head_dim) + p.nq) {
        case 33: return p8_launch<32, 1, NS>(a, p, st);
        case 34: return p8_launch<32, 2, NS>(a, p, st);
        case 65: return p8_launch<64, 1, NS>(a, p, st);
        case 66: return p8_launch<64, 2, NS>(a, p, st);
        case 129: return p8_launch<128, 1, NS>(a, p, st);
        case 130: return p8_launch<128, 2, NS>(a, p, st);
        case 193: return p8_launch<192, 1, NS>(a, p, st);
        default: return p8_launch<256, 1, NS>(a, p, st);
    }
}

}  // namespace dkv

extern "C" size_t dkv_paged8_attention_workspace(const dkv_paged8_t* cache, int32_t T, int32_t n_q_heads,
                                                 int32_t max_len) {
    if (!cache || T <= 0 || n_q_heads <= 0 || max_len <= 0 || cache->n_kv_heads <= 0 || cache->head_dim <= 0 ||
        cache->batch <= 0 || n_q_heads % cache->n_kv_heads)
        return 0;
    return dkv::p8_plan(*cache, T, n_q_heads, max_len).bytes;
}

extern "C" int dkv_paged8_attention(const dkv_paged8_t* cache, int32_t layer, const void* q, int32_t q_dtype, int32_t T,
                                    int32_t n_q_heads, const int32_t* start, const int32_t* count, int32_t max_len,
                                    void* out, void* work, size_t work_bytes, dkv_stream_t stream) {
    using namespace dkv;
    int rc = p8_check(cache, layer, "dkv_paged8_attention");
    if (rc) return rc;
    DKV_REQUIRE(q && start && out, "dkv_paged8_attention: NULL argument");
    DKV_REQUIRE(q_dtype == DKV_F32 || q_dtype == DKV_BF16, "dkv_paged8_attention: bad query dtype");
    const dkv_paged8_t c = *cache;
    DKV_REQUIRE(n_q_heads > 0 && n_q_heads % c.n_kv_heads == 0,
                "dkv_paged8_attention: query heads must be a multiple of KV heads");
    DKV_REQUIRE(max_len > 0, "dkv_paged8_attention: max_len must be > 0");
    if (T <= 0) return DKV_OK;
    if ((rc = p8_check_hot(c, T, "dkv_paged8_attention"))) return rc;
    const P8Plan p = p8_plan(c, T, n_q_heads, max_len);
    DKV_REQUIRE(p.n_chunks < 65535, "dkv_paged8_attention: max_len too large");
    DKV_REQUIRE((int64_t)c.batch * T * n_q_heads < (1LL << 31), "dkv_paged8_attention: too many rows");
    if (p.bytes && (!work || work_bytes < p.bytes || reinterpret_cast<uintptr_t>(work) % 16))
        return fail(DKV_EWORKSPACE, "dkv_paged8_attention: workspace too small or not 16-byte aligned (need " +
                                        std::to_string(p.bytes) + ")");
    P8Args a = {};
    a.c = c, a.layer = layer, a.T = T, a.Hq = n_q_heads;
    a.in_ring = p8_in_ring(c, T);
    a.n_chunks = p.n_chunks, a.per_slot = p.per_slot, a.direct = p.direct;
    a.q = q, a.start = start, a.count = count, a.out = out;
    a.qscale = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(c.head_dim)));
    a.part = static_cast<float*>(work);
    a.ml = reinterpret_cast<float2*>(a.part + (int64_t)c.batch * T * n_q_heads * (p.n_chunks + 1) * p8_dp(c.head_dim));
    return q_dtype == DKV_BF16 ? p8_launch_ns<1>(a, p, as_stream(stream)) : p8_launch_ns<3>(a, p, as_stream(stream));
}
