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
// split into three bf16 parts (NS = 3: 24 bits, as much as float32 has); bf16 queries are whole (NS = 1), and their
// probabilities two parts (PS = 2): 2^-16 of each, far below the rounding of a bf16 output. (One part, 2^-8 of each,
// put 40 % on the error of a result: 0.0023 of its norm where the output's own rounding is 0.0017.)
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

// bf16 parts of a probability, by those of a query
__host__ __device__ constexpr int p8_prob_parts(int ns) { return ns == 1 ? 2 : ns; }

constexpr int P8_MAX_LEN = 65534 * 2048;   // (chunks and the rows' own blocks are a grid's z)
constexpr int P8_UNIT = 256, P8_CHUNK = 2048, P8_UNITS = P8_CHUNK / P8_UNIT;

struct P8Args {
    dkv_paged8_t c;
    int layer, T, Hq;
    bool in_ring;
    int n_chunks;            // chunks that max_len reaches into; slot n_chunks is the rows' own blocks
    int per_slot;            // chunks per workgroup
    int bshift;              // log2(block_size)
    const void* q;
    const int32_t* start;
    const int32_t* count;
    float qscale;            // log2(e) / sqrt(head_dim)
    float* part;             // o [row][n_chunks + 1][DP]
    float2* ml;              // (m, l) [row][n_chunks + 1]
    void* out;
    bool vec;                // rows of q and out in whole, 16-byte aligned runs of 8
    bool direct;             // each row's keys all lie in one workgroup, which writes out itself
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

// A wave-uniform pointer into global memory, from the lane that holds it (a generic one would load through flat
// instructions, which wait for LDS too).
typedef const uint8_t __attribute__((address_space(1))) * p8_global;
__device__ __forceinline__ p8_global p8_lane_ptr(uint64_t addr, int lane) {
    const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)addr, lane);
    const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(addr >> 32), lane);
    return reinterpret_cast<p8_global>(hi << 32 | lo);
}
template <class V>
__device__ __forceinline__ V p8_global_load(p8_global p, int64_t off) {
    return *reinterpret_cast<const V __attribute__((address_space(1)))*>(p + off);
}

// Two tiles (32 keys) as a lane holds them: codes, or bf16 rows.
template <int DP>
struct P8Codes {
    static constexpr int PW = DP < 64 ? DP : 64, PB = PW / 4, NP = DP / PW, NW = PB / 4;
    uint32_t k[2][NP][NW], v[2][NP][NW];
    float sk[2], sv[2];
    __device__ __forceinline__ void load_k(int a, p8_global tile, uint32_t scales, int lane) {
        load_half(k[a], tile, lane);
        sk[a] = p8_scale(scales & 0xff);
    }
    __device__ __forceinline__ void load_v(int a, p8_global tile, uint32_t scales, int lane) {
        load_half(v[a], tile + 16 * DP, lane);
        sv[a] = p8_scale(scales >> 8 & 0xff);
    }
    __device__ __forceinline__ static void load_half(uint32_t (&o)[NP][NW], p8_global p, int lane) {
        typedef uint32_t vec __attribute__((ext_vector_type(NW)));
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const vec w = p8_global_load<vec>(p, i * 16 * PW + lane * PB);
#pragma unroll
            for (int j = 0; j < NW; ++j) o[i][j] = w[j];
        }
    }
    // A operand of k-step st of tile a
    __device__ __forceinline__ p8_bf16x8 kop(int a, int st) const {
        const int i = st * 32 / PW, w = st * 32 % PW / 16;
        return p8_operand(p8_words(k[a][i][w], sk[a]), p8_words(k[a][i][w + 1], sk[a]));
    }
    // A operand of d-tile dt: keys 4 q .. of tile 0, then of tile 1
    __device__ __forceinline__ p8_bf16x8 vop(int dt) const {
        const int i = dt * 16 / PW, w = dt * 16 % PW / 16;
        return p8_operand(p8_words(v[0][i][w], sv[0]), p8_words(v[1][i][w], sv[1]));
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
    __device__ __forceinline__ p8_bf16x8 vop(int dt) const {
        const int i = dt * 16 / PW, w = dt * 16 % PW / 8;
        return p8_operand(make_uint2(v[0][i][w], v[0][i][w + 1]), make_uint2(v[1][i][w], v[1][i][w + 1]));
    }
};

// Where a unit's tiles lie: lane % 16 has tile lane % 16 (tiles past the last key repeat its tile).
struct P8Unit {
    int64_t id;       // its block
    uint64_t addr;
    uint32_t sc;      // its two scale bytes
    // The three loads one behind another, apart so that a loop can issue each a unit ahead: block ids, then scales.
    __device__ __forceinline__ void find(const P8Args& A, const P8Rows& R, int k0, int k1, int lane) {
        const int mine = min(k0 + 16 * (lane % 16), k1 - 1);
        id = A.c.block_table[((int64_t)R.s * A.c.n_layers + A.layer) * A.c.max_blocks + (mine >> A.bshift)];
    }
    template <int DP>
    __device__ __forceinline__ void open(const P8Args& A, const P8Rows& R, int k0, int k1, int lane) {
        const int mine = min(k0 + 16 * (lane % 16), k1 - 1) & ((1 << A.bshift) - 1);
        const int64_t tiles = (int64_t)A.c.n_kv_heads << A.bshift;   // x 2 DP bytes
        const uint64_t blk = reinterpret_cast<uint64_t>(A.c.pool) + id * (tiles * 2 * DP + (2 * A.c.n_kv_heads + 15) / 16 * 16);
        addr = blk + (((int64_t)R.h << A.bshift) + (mine & -16)) * 2 * DP;
        sc = p8_global_load<uint16_t>(reinterpret_cast<p8_global>(blk), tiles * 2 * DP + 2 * R.h);
    }
};

// The queries of NQ q-tiles: in registers, or (QL) in LDS, for waves that share their rows.
template <int NQ, int NSTEP, int NS, bool QL>
struct P8Query {
    p8_bf16x8 q[NQ][NSTEP][NS];
    __device__ __forceinline__ void again() {}
    __device__ __forceinline__ p8_bf16x8 get(int i, int st, int j) const { return q[i][st][j]; }
    __device__ __forceinline__ void put(int i, int st, const p8_bf16x8 (&v)[NS]) {
#pragma unroll
        for (int j = 0; j < NS; ++j) q[i][st][j] = v[j];
    }
};
template <int NQ, int NSTEP, int NS>
struct P8Query<NQ, NSTEP, NS, true> {
    p8_bf16x8* lds;   // the lane's own: operand (i, st, j) at 64 ((i NSTEP + st) NS + j)
    uint32_t zero = 0;
    // (to be read again: the compiler would keep the operands in the registers that LDS is to spare)
    __device__ __forceinline__ void again() { asm volatile("" : "+v"(zero)); }
    __device__ __forceinline__ p8_bf16x8 get(int i, int st, int j) const { return lds[zero + ((i * NSTEP + st) * NS + j) * WAVE]; }
    __device__ __forceinline__ void put(int i, int st, const p8_bf16x8 (&v)[NS]) {
#pragma unroll
        for (int j = 0; j < NS; ++j) lds[((i * NSTEP + st) * NS + j) * WAVE] = v[j];
    }
};

// NQ q-tiles of 16 rows (row r0 + 16 i + lane % 16) and their softmax state.
template <int DP, int NQ, int NS, bool QL>
struct P8State {
    static constexpr int NSTEP = DP / 32, NDT = DP / 16, PS = p8_prob_parts(NS);
    P8Query<NQ, NSTEP, NS, QL> q;
    p8_f32x4 acc[NQ][NDT];
    float m[NQ], l[NQ];      // l: the lane's own keys
    int lim[NQ], last[NQ];   // the row's block start, its position

    __device__ __forceinline__ void load_limits(const P8Args& A, const P8Rows& R, int r0, int lane) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) last[i] = R.pos(r0 + 16 * i + lane % 16, A.c.block_size, lim[i]);
    }
    // k-steps st0, st0 + inc, ... of the queries
    __device__ __forceinline__ void load_rows(const P8Args& A, const P8Rows& R, int r0, int lane, int st0 = 0, int inc = 1) {
        constexpr int PW = DP < 64 ? DP : 64, PB = PW / 4;
        const int D = A.c.head_dim, col = lane % 16, g = lane / 16;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int64_t at = R.row(min(r0 + 16 * i + col, R.n_rows - 1), A.Hq) * D;
#pragma unroll
            for (int st = 0; st < NSTEP; ++st) {
                if (st % inc != st0) continue;
                const int d0 = st * 32 / PW * PW + g * PB + st * 32 % PW / 32 * 8;
                p8_bf16x8 v[NS];
                if (A.vec) {   // (D a multiple of 8 and aligned rows)
                    if constexpr (NS == 1) {
                        v[0] = __builtin_bit_cast(p8_bf16x8, d0 < D ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(A.q) + at + d0)
                                                                    : make_uint4(0, 0, 0, 0));
                    } else {
                        const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
                        const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(A.q) + at + d0);
                        const float4 a = d0 < D ? f[0] : z, b = d0 < D ? f[1] : z;
                        p8_split<NS>(a.x * A.qscale, a.y * A.qscale, v, 0);
                        p8_split<NS>(a.z * A.qscale, a.w * A.qscale, v, 2);
                        p8_split<NS>(b.x * A.qscale, b.y * A.qscale, v, 4);
                        p8_split<NS>(b.z * A.qscale, b.w * A.qscale, v, 6);
                    }
                } else {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[e] = d0 + e >= D ? 0.0f : NS == 1 ? bf16_to_f32(static_cast<const uint16_t*>(A.q)[at + d0 + e])
                                                            : static_cast<const float*>(A.q)[at + d0 + e] * A.qscale;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) p8_split<NS>(x[e], x[e + 1], v, e);
                }
                q.put(i, st, v);
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

    // scores of the 32 keys of x, to be scaled (bf16 queries enter the products as they are, float32 ones scaled)
    template <class Keys>
    __device__ __forceinline__ void scores(const Keys& x, float (&p)[NQ][8]) {
        p8_f32x4 s[NQ][2];
        q.again();
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
                    for (int j = 0; j < NS; ++j) s[i][a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kv, q.get(i, st, j), s[i][a], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) p[i][k] = s[i][k / 4][k % 4];
    }
    // Scores to probabilities against the row's reference m, the maximum of the first keys that it saw, moved (and its
    // sums with it) only when a score is more than 2^8 times as likely: a maximum that moves with every record would
    // have the 16 rows rescale their sums in almost every one of a unit's eight steps. The reference is a function of
    // the row's own scores, and a probability of up to 256 is as exact as one of up to 1.
    __device__ __forceinline__ void softmax(float (&p)[NQ][8], p8_bf16x8 (&ph)[NQ][PS], float qscale) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            float mx = p[i][0];
#pragma unroll
            for (int k = 1; k < 8; ++k) mx = fmaxf(mx, p[i][k]);
            mx = lanegroup_max(mx);
            if constexpr (NS == 1) mx *= qscale;
            const float mo = m[i];
            if (__any(mx > mo + 8.0f)) {   // (-inf + 8 < mx: the first keys)
                const float mn = mx > mo + 8.0f ? mx : mo;
                const float a = mn == mo ? 1.0f : exp2_hw(mo - mn);
                m[i] = mn;
                l[i] *= a;
                if (__any(a != 1.0f && mo != -INFINITY)) {
#pragma unroll
                    for (int dt = 0; dt < NDT; ++dt) acc[i][dt] *= a;
                }
            }
            const float ms = m[i] == -INFINITY ? 0.0f : m[i];   // a row that sees no key yet: p = 0
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                p[i][k] = exp2_hw(NS == 1 ? fmaf(p[i][k], qscale, -ms) : p[i][k] - ms);
                sum += p[i][k];
            }
            l[i] += sum;
#pragma unroll
            for (int k = 0; k < 8; k += 2) p8_split<PS>(p[i][k], p[i][k + 1], ph[i], k);
        }
    }
    // O^T += V^T . P^T of keys that some rows do not see (their P is 0, and 0 * NaN is NaN): what is not finite in V
    // stays out of the product, and then, rarely, marks the channels of the rows that do see it. vis: the lane's keys'
    // bits of its row.
    template <class Keys>
    __device__ __forceinline__ void values_masked(const Keys& x, const p8_bf16x8 (&ph)[NQ][PS], const uint32_t (&vis)[NQ]) {
        auto odd = [](uint32_t u) {   // a mask of the halves that are no finite bf16
            return ((u & 0x7f80) == 0x7f80 ? 0xffffu : 0u) | ((u & 0x7f800000) == 0x7f800000 ? 0xffff0000u : 0u);
        };
        uint32_t any = 0;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            uint4 w = __builtin_bit_cast(uint4, x.vop(dt));
            const uint4 b = make_uint4(odd(w.x), odd(w.y), odd(w.z), odd(w.w));
            any |= b.x | b.y | b.z | b.w;
            w.x &= ~b.x, w.y &= ~b.y, w.z &= ~b.z, w.w &= ~b.w;
#pragma unroll
            for (int i = 0; i < NQ; ++i)
#pragma unroll
                for (int j = 0; j < PS; ++j)
                    acc[i][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(p8_bf16x8, w), ph[i][j], acc[i][dt], 0, 0, 0);
        }
        if (!__any(any != 0)) return;
        // counts of the +inf, -inf and NaN that a row sees, per channel: products of ones
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            uint4 see;
            uint32_t* sw = &see.x;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                sw[k] = ((vis[i] >> 2 * k & 1) ? 0x3f80u : 0u) | ((vis[i] >> (2 * k + 1) & 1) ? 0x3f800000u : 0u);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                const uint4 w = __builtin_bit_cast(uint4, x.vop(dt));
                auto ones = [&](auto is) {
                    auto f = [&](uint32_t u) { return (is(u & 0xffff) ? 0x3f80u : 0u) | (is(u >> 16) ? 0x3f800000u : 0u); };
                    const p8_bf16x8 v = __builtin_bit_cast(p8_bf16x8, make_uint4(f(w.x), f(w.y), f(w.z), f(w.w)));
                    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(p8_bf16x8, see), p8_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                };
                const p8_f32x4 up = ones([](uint32_t h) { return h == 0x7f80; }), down = ones([](uint32_t h) { return h == 0xff80; });
                const p8_f32x4 none = ones([](uint32_t h) { return (h & 0x7fff) > 0x7f80; });
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float t = acc[i][dt][e];
                    if (up[e] > 0.0f) t += INFINITY;
                    if (down[e] > 0.0f) t -= INFINITY;
                    if (none[e] > 0.0f) t = __uint_as_float(0x7fc00000);
                    acc[i][dt][e] = t;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // The keys of x, from kb on; next_k is called once K is used, which may then hold the next step's. Without MASK
    // every row sees both tiles; with it all of a tile or none, keys below lim.
    template <bool MASK, class Keys, class Next>
    __device__ __forceinline__ void step(const Keys& x, int kb, float qscale, Next next_k) {
        float p[NQ][8];
        p8_bf16x8 ph[NQ][PS];
        scores(x, p);
        next_k();
        uint32_t vis[NQ];
        if constexpr (MASK) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                vis[i] = (kb < lim[i] ? 0xfu : 0u) | (kb + 16 < lim[i] ? 0xf0u : 0u);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (!(vis[i] >> k & 1)) p[i][k] = -INFINITY;
            }
        }
        softmax(p, ph, qscale);
        if constexpr (MASK) return values_masked(x, ph, vis);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            const p8_bf16x8 v = x.vop(dt);
#pragma unroll
            for (int i = 0; i < NQ; ++i)
#pragma unroll
                for (int j = 0; j < PS; ++j) acc[i][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, ph[i][j], acc[i][dt], 0, 0, 0);
        }
    }
    // The rows' own blocks: keys lim <= k <= last. past: the first position that holds no row (stale memory from there).
    __device__ __forceinline__ void step_own(P8Bf16<DP>& x, int kb, int past, float qscale, int lane) {
        constexpr int NW = P8Bf16<DP>::NW, NP = P8Bf16<DP>::NP;
        const int g = lane / 16;
        float p[NQ][8];
        p8_bf16x8 ph[NQ][PS];
        scores(x, p);
        uint32_t vis[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            vis[i] = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int key = kb + k / 4 * 16 + 4 * g + k % 4;
                if (key < lim[i] || key > last[i]) p[i][k] = -INFINITY;
                else vis[i] |= 1u << k;
            }
        }
        softmax(p, ph, qscale);
        if (kb + 32 > past) {   // (V: two keys per word)
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int i = 0; i < NP; ++i)
#pragma unroll
                    for (int w = 0; w < NW; ++w) {
                        const int key = kb + 16 * a + 4 * g + 2 * (w % 2);
                        x.v[a][i][w] &= key >= past ? 0u : key + 1 >= past ? 0xffffu : ~0u;
                    }
        }
        values_masked(x, ph, vis);
    }

    // The sealed keys [k0, k1), k0 a unit's start, k1 at most its end; u holds their tiles. Keys below `all` are seen by
    // every row. The next step's K is fetched once this step's scores are there, its V once this step's V is used: with
    // one set of registers (SETS = 1: two sets are 32 more, which spill beside two q-tiles) half a step ahead, with two
    // a step and a half.
    template <int SETS>
    __device__ __forceinline__ void unit(const P8Args& A, const P8Unit& u, int k0, int k1, int all, int lane) {
        P8Codes<DP> x[SETS];
        const int steps = (k1 - k0 + 31) / 32;
        auto fetch_k = [&](P8Codes<DP>& c, int j) {
#pragma unroll
            for (int a = 0; a < 2; ++a) c.load_k(a, p8_lane_ptr(u.addr, 2 * j + a), __builtin_amdgcn_readlane((int)u.sc, 2 * j + a), lane);
        };
        auto fetch_v = [&](P8Codes<DP>& c, int j) {
#pragma unroll
            for (int a = 0; a < 2; ++a) c.load_v(a, p8_lane_ptr(u.addr, 2 * j + a), __builtin_amdgcn_readlane((int)u.sc, 2 * j + a), lane);
        };
#pragma unroll
        for (int i = 0; i < SETS; ++i) {
            fetch_k(x[i], min(i, steps - 1));
            fetch_v(x[i], min(i, steps - 1));
        }
        const int whole = max(0, min((all - k0) / 32, steps)) / SETS * SETS;   // steps that every row sees
#pragma nounroll
        for (int j = 0; j < whole; j += SETS) {
#pragma unroll
            for (int i = 0; i < SETS; ++i) {
                const int nj = min(j + i + SETS, steps - 1);
                step<false>(x[i], k0 + 32 * (j + i), A.qscale, [&]() { fetch_k(x[i], nj); });
                fetch_v(x[i], nj);
            }
        }
#pragma nounroll
        for (int j = whole; j < steps; j += SETS) {
#pragma unroll
            for (int i = 0; i < SETS; ++i) {
                const int nj = min(j + i + SETS, steps - 1);
                if (j + i < steps) step<true>(x[i], k0 + 32 * (j + i), A.qscale, [&]() { fetch_k(x[i], nj); });
                fetch_v(x[i], nj);
            }
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

__device__ __forceinline__ uint32_t p8_bf16_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((p8_f32x2){a, b}, p8_bf16x2));
}

// a row's four channels from d0 of its result; l of the row
template <int NS>
__device__ __forceinline__ void p8_store_out(const P8Args& A, int64_t row, int d0, p8_f32x4 o, float l) {
    const int D = A.c.head_dim;
    if (A.vec) {
        if (d0 >= D) return;
        if constexpr (NS == 1)
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(A.out) + row * D + d0) =
                make_uint2(p8_bf16_pair(o[0] / l, o[1] / l), p8_bf16_pair(o[2] / l, o[3] / l));
        else
            *reinterpret_cast<p8_f32x4*>(static_cast<float*>(A.out) + row * D + d0) = p8_f32x4{o[0] / l, o[1] / l, o[2] / l, o[3] / l};
        return;
    }
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

// ---------------------------------------------------------------- few rows: a workgroup streams its chunks
// Two float32 q-tiles' queries of 128 channels would take 96 registers of the 256 that two waves per SIMD have, bf16 ones
// 32 that spill; the eight waves share them in LDS instead (5 rows of 4 heads each, batch 32, context 32k, bf16, with one
// part of the probabilities: 502 us with registers, 465 so).
__host__ __device__ constexpr bool p8_query_in_lds(int dp, int nq, int ns) { return nq * (dp / 32) * ns > 16 || nq * (dp / 32) >= 8; }
__host__ __device__ constexpr size_t p8_chunk_lds(int dp, int nq, int ns) {
    return (size_t)P8_UNITS * nq * ((dp / 16) * 1024 + 16 * sizeof(float2)) +
           (p8_query_in_lds(dp, nq, ns) ? (size_t)nq * (dp / 32) * ns * 1024 : 0);
}
// Grid (KV head x sequence, q-group, run of chunks or own blocks). Eight waves, one unit of a chunk each, straight from
// memory to registers; their states meet in LDS and leave as the chunk's. Bound by memory: 32 sequences of 32700 tokens, 8
// KV heads of 128, one token each, bf16, 383 us (5.6 TB/s), float32 403; 5 rows of 4 heads each, bf16, 472, float32 (three
// products for one, on 32 rows for 20: 295 us of matrix instructions) 505 to 540.
// ONE: all keys lie in one chunk, and the workgroup takes the rows' own blocks too (its last wave, which few contexts
// give a unit) and writes out: the merge would cost as much again as a short context's attention.
template <int DP, int NQ, int NS, bool ONE>
__global__ void __launch_bounds__(512) paged8_chunk_kernel(P8Args A) {
    // (two sets of codes where they do not spill: 16 / 8 heads of 256, 16 x 16000 keys, float32, 5 rows 420 us with two, 247
    // with one; of 192 bf16 200 and 157)
    constexpr int NDT = DP / 16, SETS = DP <= 64 || (NQ == 1 && DP <= 128) ? 2 : 1;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const P8Rows R = p8_rows(A, blockIdx.x);
    const int r0 = blockIdx.y * 16 * NQ, bs = A.c.block_size;
    if (R.len <= R.s0) {
        if (blockIdx.z == 0) p8_zero_rows<NS>(A, R, r0, r0 + 16 * NQ, threadIdx.x, 512);
        return;
    }
    int lim0, lim1;
    R.pos(r0, bs, lim0);                                               // the least and the largest of the rows'
    const int last1 = R.pos(r0 + 16 * NQ - 1, bs, lim1);
    const bool own = !ONE && blockIdx.z == gridDim.z - 1;              // this workgroup takes the rows' own blocks
    const int ch0 = blockIdx.z * A.per_slot;
    const int ch1 = ONE || own ? ch0 + 1 : min(min(ch0 + A.per_slot, A.n_chunks), (lim1 + P8_CHUNK - 1) / P8_CHUNK);
    if (ch0 >= ch1) return;
    extern __shared__ __align__(16) char p8_lds[];
    constexpr bool QL = p8_query_in_lds(DP, NQ, NS);
    p8_f32x4* so = reinterpret_cast<p8_f32x4*>(p8_lds);                // [units][NQ][NDT][64]
    float2* sml = reinterpret_cast<float2*>(p8_lds + P8_UNITS * NQ * NDT * 1024);   // [units][NQ][16]
    // the wave's unit of the next chunk is looked up while this one's keys stream
    P8Unit u = {}, nu = {};
    int k0 = ch0 * P8_CHUNK + wave * P8_UNIT;
    if (!own && k0 < lim1) u.find(A, R, k0, min(k0 + P8_UNIT, lim1), lane);
    P8State<DP, NQ, NS, QL> st;
    if constexpr (QL) {   // (the waves share the rows: each splits its part of the k-steps)
        st.q.lds = reinterpret_cast<p8_bf16x8*>(p8_lds + P8_UNITS * NQ * (NDT * 1024 + 16 * sizeof(float2))) + lane;
        st.load_rows(A, R, r0, lane, wave, 8);
        __syncthreads();
    } else {
        st.load_rows(A, R, r0, lane);
    }
    st.load_limits(A, R, r0, lane);
    if (!own && k0 < lim1) u.template open<DP>(A, R, k0, min(k0 + P8_UNIT, lim1), lane);
    auto leave = [&](int slot) {   // this wave's state
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            if (lane < 16) sml[(slot * NQ + i) * 16 + lane] = make_float2(st.m[i], st.l[i]);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) so[((slot * NQ + i) * NDT + dt) * WAVE + lane] = st.acc[i][dt];
        }
    };
    // d-tile x / 64 (of all q-tiles), lane x % 64 of the sums: slots 0 .. n - 1 in order behind (m, l, o)
    auto fold = [&](int x, int n, float& m, float& l, p8_f32x4& o) {
        for (int w = 0; w < n; ++w) {
            const float2 ml = sml[(w * NQ + x / WAVE / NDT) * 16 + x % 16];
            const p8_f32x4 ou = so[w * NQ * NDT * WAVE + x];
            float a, b;
            m = fold_max(m, ml.x, a, b);
            l = fold_sum(l, a, ml.y, b);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fold_sum(o[e], a, ou[e], b);
        }
    };
    if constexpr (ONE) {
        const int units = min(P8_UNITS, (lim1 + P8_UNIT - 1) / P8_UNIT);   // (longer than max_len said: its first keys)
        if (wave < units) {
            st.clear();
            st.template unit<SETS>(A, u, k0, min(k0 + P8_UNIT, lim1), lim0, lane);
            leave(wave);
        }
        if (wave == P8_UNITS - 1) {
            st.clear();
            st.own_blocks(A, R, lim0, last1, lane);
        }
        __syncthreads();
        constexpr int NI = (NQ * NDT * WAVE + 511) / 512;
        float m[NI], l[NI];
        p8_f32x4 o[NI];
#pragma unroll
        for (int y = 0; y < NI; ++y) {
            const int x = threadIdx.x + 512 * y;
            m[y] = -INFINITY, l[y] = 0.0f, o[y] = p8_f32x4{0.f, 0.f, 0.f, 0.f};
            if (x < NQ * NDT * WAVE) fold(x, units, m[y], l[y], o[y]);
        }
        __syncthreads();
        if (wave == P8_UNITS - 1) leave(0);
        __syncthreads();
#pragma unroll
        for (int y = 0; y < NI; ++y) {
            const int x = threadIdx.x + 512 * y, r = r0 + 16 * (x / WAVE / NDT) + x % 16;
            if (x >= NQ * NDT * WAVE || r >= R.n_rows) continue;
            fold(x, 1, m[y], l[y], o[y]);
            p8_store_out<NS>(A, R.row(r, A.Hq), x / WAVE % NDT * 16 + x % WAVE / 16 * 4, o[y], l[y]);
        }
        return;
    }
    for (int ch = ch0; ch < ch1; ++ch, k0 += P8_CHUNK) {
        const int units = own ? 1 : min(P8_UNITS, (lim1 - ch * P8_CHUNK + P8_UNIT - 1) / P8_UNIT);
        if (wave < units) {
            const int n0 = k0 + P8_CHUNK, n1 = min(n0 + P8_UNIT, lim1);
            const bool more = ch + 1 < ch1 && n0 < lim1;
            if (more) nu.find(A, R, n0, n1, lane);
            st.clear();
            if (own) st.own_blocks(A, R, lim0, last1, lane);
            else st.template unit<SETS>(A, u, k0, min(k0 + P8_UNIT, lim1), lim0, lane);
            if (more) {
                nu.template open<DP>(A, R, n0, n1, lane);
                u = nu;
            }
            leave(wave);
        }
        __syncthreads();
        for (int x = threadIdx.x; x < NQ * NDT * WAVE; x += 512) {
            const int ln = x % WAVE, r = r0 + 16 * (x / WAVE / NDT) + ln % 16;
            if (r >= R.n_rows) continue;
            float m = -INFINITY, l = 0.0f;
            p8_f32x4 o = {0.f, 0.f, 0.f, 0.f};
            fold(x, units, m, l, o);
            const int64_t slot = R.row(r, A.Hq) * (A.n_chunks + 1) + (own ? A.n_chunks : ch);
            const int dt = x / WAVE % NDT;
            *reinterpret_cast<p8_f32x4*>(A.part + slot * DP + dt * 16 + ln / 16 * 4) = o;
            if (dt == 0 && ln < 16) A.ml[slot] = make_float2(m, l);
        }
        if (ch + 1 < ch1) __syncthreads();
    }
}

// ---------------------------------------------------------------- many rows: the waves walk the keys together
// Grid (KV head x sequence, q-group, slot). NW waves with NQ q-tiles each. Every 32 keys are converted to bf16 once per
// workgroup, into LDS in operand order, two stages deep with the next step's codes in registers: a wave's own
// conversion (64 instructions a step) would cost as much as half its softmax, and its loads 8 KB of L1 each. Of a
// wave's state the unit's and the chunk's sums are registers, the sums over the chunks before lie in LDS (touched once
// in 2048 keys). A prompt of 4096 tokens, 32 / 8 heads of 128: bf16 266 us (517 TFLOP/s; with one part of the
// probabilities, a third fewer products, 225), float32 425 to 443. A step of 32 keys takes 1.5 us in bf16 where its
// products alone take 0.6: the eight waves come to their products, their exponentials and
// their LDS reads together, and registers leave no room to run one step's products under another's softmax.
template <int DP>
struct P8Staged {
    const char* k;   // the lane's own: operand (a, st) at 1024 (a NSTEP + st)
    const char* v;   // operand dt at 1024 dt: keys of tile 0, then of tile 1
    __device__ __forceinline__ p8_bf16x8 kop(int a, int st) const {
        return *reinterpret_cast<const p8_bf16x8*>(k + 1024 * (a * (DP / 32) + st));
    }
    __device__ __forceinline__ p8_bf16x8 vop(int dt) const { return *reinterpret_cast<const p8_bf16x8*>(v + 1024 * dt); }
};

template <int DP, int NQ, int NS, int NW>
__global__ void __launch_bounds__(64 * NW, 1) paged8_walk_kernel(P8Args A) {
    constexpr int NSTEP = DP / 32, NDT = DP / 16, PW = DP < 64 ? DP : 64, PB = PW / 4, NP = DP / PW, NWD = PB / 4;
    constexpr int PIECES = 4 * NP;                          // (tile, K or V, panel) of a step, one per wave and turn
    constexpr int TURNS = (PIECES + NW - 1) / NW;
    constexpr int STAGE = 2 * 32 * DP * 2;                  // bytes: K, V of 32 keys
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const P8Rows R = p8_rows(A, blockIdx.x);
    const int qg = gridDim.y - 1 - blockIdx.y;   // the last rows see the most keys and go first
    const int w0 = qg * NW * 16 * NQ, r0 = w0 + wave * 16 * NQ, bs = A.c.block_size;
    if (R.len <= R.s0) {
        if (blockIdx.z == 0) p8_zero_rows<NS>(A, R, w0, w0 + NW * 16 * NQ, threadIdx.x, 64 * NW);
        return;
    }
    int lim0, lim1, limw;   // of the wave's rows, and the largest of the workgroup's
    R.pos(r0, bs, lim0);
    const int last1 = R.pos(r0 + 16 * NQ - 1, bs, lim1);
    R.pos(w0 + NW * 16 * NQ - 1, bs, limw);
    const bool live = r0 < R.n_rows;
    const bool own = A.direct || blockIdx.z == gridDim.z - 1;   // this workgroup takes the rows' own blocks
    const int ch0 = A.direct ? 0 : blockIdx.z * A.per_slot;
    const int ch1 = A.direct ? A.n_chunks : own ? ch0 : min(ch0 + A.per_slot, A.n_chunks);
    const int kbeg = ch0 * P8_CHUNK, kend = own && !A.direct ? kbeg : min(ch1 * P8_CHUNK, limw);
    if (!own && kbeg >= limw) return;
    extern __shared__ __align__(16) char p8_lds[];
    p8_f32x4* so = reinterpret_cast<p8_f32x4*>(p8_lds + 2 * STAGE) + (int64_t)wave * NQ * NDT * WAVE + lane;

    P8State<DP, NQ, NS, false> st;
    st.load_rows(A, R, r0, lane);
    st.load_limits(A, R, r0, lane);
    p8_f32x4 oc[NQ][NDT];                      // the chunk's units so far
    float mc[NQ], lc[NQ], mt[NQ], lt[NQ];      // (t: the chunks so far)
    auto clear_chunk = [&]() {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            mc[i] = -INFINITY, lc[i] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) oc[i][dt] = p8_f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    auto fold_unit = [&]() {
        st.end_unit();
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            float a, b;
            mc[i] = fold_max(mc[i], st.m[i], a, b);
            lc[i] = fold_sum(lc[i], a, st.l[i], b);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
                for (int e = 0; e < 4; ++e) oc[i][dt][e] = fold_sum(oc[i][dt][e], a, st.acc[i][dt][e], b);
        }
        st.clear();
    };
    // (m, l, o) into the sums over the chunks
    auto fold_total = [&](const float (&m)[NQ], const float (&l)[NQ], const p8_f32x4 (&o)[NQ][NDT]) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            float a, b;
            mt[i] = fold_max(mt[i], m[i], a, b);
            lt[i] = fold_sum(lt[i], a, l[i], b);
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
                p8_f32x4 t = so[(i * NDT + dt) * WAVE];
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = fold_sum(t[e], a, o[i][dt][e], b);
                so[(i * NDT + dt) * WAVE] = t;
            }
        }
    };
    auto store_part = [&](int slot, const float (&m)[NQ], const float (&l)[NQ], const p8_f32x4 (&o)[NQ][NDT]) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int r = r0 + 16 * i + lane % 16;
            if (r >= R.n_rows) continue;
            const int64_t ps = R.row(r, A.Hq) * (A.n_chunks + 1) + slot;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt)
                *reinterpret_cast<p8_f32x4*>(A.part + ps * DP + dt * 16 + lane / 16 * 4) = o[i][dt];
            if (lane < 16) A.ml[ps] = make_float2(m[i], l[i]);
        }
    };
    if (A.direct) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            mt[i] = -INFINITY, lt[i] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) so[(i * NDT + dt) * WAVE] = p8_f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    clear_chunk();
    st.clear();

    const int steps = (kend - kbeg + 31) / 32;
    typedef uint32_t vec __attribute__((ext_vector_type(NWD)));
    vec pre[TURNS];          // the codes of the step after the next, and their scales
    float psc[TURNS];
    // the unit being fetched and the one after it (its blocks found, then opened, a unit ahead)
    P8Unit u = {}, nu = {};
    auto fetch = [&](int j) {
        const int kb = kbeg + 32 * j;
        if (j % (P8_UNIT / 32) == 0) {
            u.addr = nu.addr, u.sc = nu.sc;
            if (kb + P8_UNIT < kend) nu.find(A, R, kb + P8_UNIT, kend, lane);
        } else if (j % (P8_UNIT / 32) == 4) {
            const int kn = kb / P8_UNIT * P8_UNIT + P8_UNIT;
            if (kn < kend) nu.template open<DP>(A, R, kn, kend, lane);
        }
#pragma unroll
        for (int x = 0; x < TURNS; ++x) {
            const int pc = wave + x * NW;   // panel, K or V, tile
            if (PIECES % NW && pc >= PIECES) break;
            const int t = 2 * (j % (P8_UNIT / 32)) + pc / (2 * NP), kv = pc / NP % 2, i = pc % NP;
            pre[x] = p8_global_load<vec>(p8_lane_ptr(u.addr, t), (kv * DP + i * PW) * 16 + lane * PB);
            psc[x] = p8_scale((uint32_t)__builtin_amdgcn_readlane((int)u.sc, t) >> 8 * kv & 0xff);
        }
    };
    auto stage = [&](int j) {   // the fetched codes into stage j % 2
        char* at = p8_lds + j % 2 * STAGE + lane * 16;
#pragma unroll
        for (int x = 0; x < TURNS; ++x) {
            const int pc = wave + x * NW;
            if (PIECES % NW && pc >= PIECES) break;
            const int a = pc / (2 * NP), kv = pc / NP % 2, i = pc % NP;
            if (kv == 0) {
#pragma unroll
                for (int w = 0; w < NWD; w += 2)
                    *reinterpret_cast<p8_bf16x8*>(at + 1024 * (a * NSTEP + i * (PW / 32) + w / 2)) =
                        p8_operand(p8_words(pre[x][w], psc[x]), p8_words(pre[x][w + 1], psc[x]));
            } else {
#pragma unroll
                for (int w = 0; w < NWD; ++w)
                    *reinterpret_cast<uint2*>(at + STAGE / 2 + 1024 * (i * (PW / 16) + w) + 8 * a) = p8_words(pre[x][w], psc[x]);
            }
        }
    };
    if (steps > 0) {
        nu.find(A, R, kbeg, kend, lane);
        nu.template open<DP>(A, R, kbeg, kend, lane);
        fetch(0);
        stage(0);
        fetch(min(1, steps - 1));
    }
    // (a loop over the units around those over their steps: what only a unit's end needs can leave the registers)
    constexpr int US = P8_UNIT / 32;
    int limg;   // the least lim of the workgroup's rows
    R.pos(w0, bs, limg);
    const int whole = max(0, min((limg - kbeg) / 32, steps));   // steps that every row sees
    auto next = [&](int j) {
        __syncthreads();   // stage j % 2 is whole, and every wave is done with the other
        if (j + 1 < steps) {
            stage(j + 1);
            if (j + 2 < steps) fetch(j + 2);
        }
        const char* at = p8_lds + j % 2 * STAGE + lane * 16;
        return P8Staged<DP>{at, at + STAGE / 2};
    };
    int ch = ch0;
    for (int j0 = 0; j0 < steps; j0 += US) {
        const int j1 = min(j0 + US, steps), jw = max(j0, min(j1, whole));
#pragma nounroll
        for (int j = j0; j < jw; ++j) {
            const P8Staged<DP> x = next(j);
            st.template step<false>(x, 0, A.qscale, []() {});   // (rows past the last compute as the last one does)
        }
#pragma nounroll
        for (int j = jw; j < j1; ++j) {
            const P8Staged<DP> x = next(j);
            const int kb = kbeg + 32 * j;
            if (live && kb < lim1) st.template step<true>(x, kb, A.qscale, []() {});
        }
        const int ku = kbeg + 32 * j0;
        if (!live || ku >= lim1) continue;
        fold_unit();
        if ((ku + P8_UNIT) % P8_CHUNK == 0 || ku + P8_UNIT >= lim1) {
            if (A.direct) fold_total(mc, lc, oc);
            else store_part(ch, mc, lc, oc);
            clear_chunk();
            ++ch;
        }
    }
    if (!own || !live) return;
    st.own_blocks(A, R, lim0, last1, lane);
    if (!A.direct) return store_part(A.n_chunks, st.m, st.l, st.acc);
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        float a, b;
        mt[i] = fold_max(mt[i], st.m[i], a, b);
        const float l = fold_sum(lt[i], a, st.l[i], b);
        const int r = r0 + 16 * i + lane % 16;
        if (r >= R.n_rows) continue;
        const int64_t row = R.row(r, A.Hq);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
            p8_f32x4 t = so[(i * NDT + dt) * WAVE];
#pragma unroll
            for (int e = 0; e < 4; ++e) t[e] = fold_sum(t[e], a, st.acc[i][dt][e], b);
            p8_store_out<NS>(A, row, dt * 16 + lane / 16 * 4, t, l);
        }
    }
}

// ---------------------------------------------------------------- merge
// One wave per row: its chunks in order, its own block last. Bound by its launch and one round of loads (1024 rows of 17
// slots: 8 us).
template <int DP, int NS>
__global__ void __launch_bounds__(256) paged8_merge_kernel(P8Args A) {
    constexpr int ND = (DP + WAVE - 1) / WAVE;
    const int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / WAVE;
    if (row >= (int64_t)A.c.batch * A.T * A.Hq) return;
    const int lane = threadIdx.x % WAVE, D = A.c.head_dim;
    const int s = (int)(row / A.Hq / A.T), t = (int)(row / A.Hq % A.T), s0 = A.start[s];
    const int len = s0 + p8_new_rows(A.c, A.T, s0, A.count, s), p = min(s0 + t, len - 1);
    if (len <= s0) return;   // no new rows: written
    const int lim = p & -A.c.block_size;
    const int n = min((lim + P8_CHUNK - 1) / P8_CHUNK, A.n_chunks);
    const float* po = A.part + row * (A.n_chunks + 1) * DP;
    const float2* pm = A.ml + row * (A.n_chunks + 1);
    // the row's slots: its chunks, then its own block; the loads of NB of them are in flight at once
    constexpr int NB = 8;
    float m = -INFINITY, l = 0.0f, o[ND] = {};
    for (int c0 = 0; c0 <= n; c0 += NB) {
        float2 ml[NB];
        float v[NB][ND];
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            const int slot = c0 + k < n ? c0 + k : A.n_chunks;
            ml[k] = pm[slot];
#pragma unroll
            for (int i = 0; i < ND; ++i) v[k][i] = po[(int64_t)slot * DP + min(lane + WAVE * i, D - 1)];
        }
#pragma unroll
        for (int k = 0; k < NB; ++k)
            if (c0 + k <= n) {
                float a, b;
                m = fold_max(m, ml[k].x, a, b);
                l = fold_sum(l, a, ml[k].y, b);
#pragma unroll
                for (int i = 0; i < ND; ++i) o[i] = fold_sum(o[i], a, v[k][i], b);
            }
    }
#pragma unroll
    for (int i = 0; i < ND; ++i) {
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

// waves and q-tiles of a walking workgroup: eight waves (two per SIMD) where the state fits 256 registers
__host__ constexpr int p8_walk_waves(int dp) { return dp > 128 ? 4 : 8; }
__host__ constexpr int p8_walk_tiles(int dp, int ns) { return dp > 128 || ns > 1 ? 1 : 2; }

// Which kernel, where either could take the rows: the one that a model of their times says is faster. A workgroup that
// streams a chunk needs `full` us for its 2048 keys where every CU has one, and `base` however few keys it has (half of
// that where CUs stay free); a walking one, of many more rows, 12 us and `step` per 32 keys. Measured, streaming against
// walking, us: 32 / 8 heads of 128, bf16, one sequence: 400 rows on no context 22 / 36, 1600 rows 91 / 105; on 2000 keys
// 100 rows 25 / 121, 400 rows 63 / 129, 1600 rows 231 / 206; four sequences, 400 rows on 2000 keys 202 / 163. 9 / 3
// heads of 64, float32: 400 rows on 8000 keys 60 / 84, 1600 rows 183 / 167.
static bool p8_walks(const dkv_paged8_t& c, int64_t tiles, int T, int max_len, int nq, int slots, int per_slot, int ns) {
    const int dp = p8_dp(c.head_dim), at = dp == 32 ? 0 : dp / 64;
    static const float base[2][5] = {{9, 12, 13, 13, 15}, {14, 23, 20, 18, 25}}, full[2][5] = {{12, 16, 26, 19, 24}, {19, 30, 40, 27, 36}},
                       step[2][5] = {{.9f, 1.1f, 1.75f, 1.2f, 1.5f}, {.7f, .9f, 1.45f, 1.45f, 2.2f}};
    const int64_t heads = (int64_t)c.n_kv_heads * c.batch, groups = (tiles + nq - 1) / nq;
    if (groups > 65535) return true;
    const float keys = (float)std::max(1, max_len - T / 2), chunks = keys / P8_CHUNK;   // of a row, on average
    const float f = full[ns > 1][at] * chunks, b = base[ns > 1][at];
    const float stream = std::max(std::min(std::max(f, b / 2), full[ns > 1][at]), groups * heads * std::max(f, b) / 256.0f);
    const int per = p8_walk_waves(dp) * p8_walk_tiles(dp, ns);
    const int64_t wgs = (tiles + per - 1) / per * heads * slots;
    const float longest = (float)std::min<int64_t>(max_len, (int64_t)per_slot * P8_CHUNK);
    const float walk = 12.0f + step[ns > 1][at] / 32.0f * std::max(longest, (float)((wgs + 255) / 256) * keys / slots);
    return walk < stream;
}

static P8Plan p8_plan(const dkv_paged8_t& c, int T, int Hq, int max_len, int ns) {
    P8Plan p = {};
    const int dp = p8_dp(c.head_dim);
    const int64_t rows = (int64_t)T * (Hq / c.n_kv_heads), tiles = (rows + 15) / 16;
    p.n_chunks = (max_len + P8_CHUNK - 1) / P8_CHUNK;
    p.nq = tiles > 1 && dp <= 128 ? 2 : 1;
    // slots of a walk: where its workgroups are too few for 256 CUs, the chunks go to several, their states through memory
    int slots = 1, per_slot = p.n_chunks;
    {
        const int per = p8_walk_waves(dp) * p8_walk_tiles(dp, ns);
        const int64_t wgs = (tiles + per - 1) / per * c.n_kv_heads * c.batch;
        if (wgs < 256 && p.n_chunks > 1) {
            slots = (int)std::min<int64_t>(p.n_chunks, (512 + wgs - 1) / wgs);
            per_slot = (p.n_chunks + slots - 1) / slots;
            slots = (p.n_chunks + per_slot - 1) / per_slot;
        }
    }
    p.walk = tiles > p.nq && p8_walks(c, tiles, T, max_len, p.nq, slots, per_slot, ns);
    p.slots = 1, p.per_slot = p.n_chunks, p.direct = p.walk || p.n_chunks == 1;
    if (!p.walk && !p.direct) {
        // a run of chunks per workgroup: about four workgroups per CU, as many as its chunks give
        const int64_t wgs = (tiles + p.nq - 1) / p.nq * c.n_kv_heads * c.batch;
        p.per_slot = (int)std::max<int64_t>(1, p.n_chunks * wgs / 1024);
        p.slots = (p.n_chunks + p.per_slot - 1) / p.per_slot;
    }
    if (p.walk) {
        p.nq = p8_walk_tiles(dp, ns);
        p.direct = slots == 1;
        p.slots = slots, p.per_slot = per_slot;
    }
    if (!p.direct) p.bytes = (size_t)c.batch * T * Hq * (p.n_chunks + 1) * (dp + 2) * sizeof(float);
    return p;
}

template <int DP, int NS>
static int p8_launch_walk(P8Args& a, const P8Plan& p, int64_t tiles, hipStream_t st) {
    constexpr int NW = p8_walk_waves(DP), NQ = p8_walk_tiles(DP, NS);
    const size_t lds = 2 * 2 * 32 * DP * 2 + (size_t)NW * NQ * (DP / 16) * 1024;
    const int64_t groups = (tiles + NW * NQ - 1) / (NW * NQ);
    DKV_REQUIRE(groups <= 65535, "dkv_paged8_attention: too many rows");
    auto fn = paged8_walk_kernel<DP, NQ, NS, NW>;
    static size_t done[16] = {};
    if (!reserve_lds(reinterpret_cast<const void*>(fn), lds, done))
        return fail(DKV_ELAUNCH, "dkv_paged8_attention: cannot reserve " + std::to_string(lds) + " B of LDS");
    hipLaunchKernelGGL(fn, dim3(a.c.n_kv_heads * a.c.batch, (int)groups, p.direct ? 1 : p.slots + 1), dim3(64 * NW), lds, st, a);
    return DKV_OK;
}

template <int DP, int NQ, int NS, bool ONE>
static int p8_launch_chunk(P8Args& a, const P8Plan& p, int64_t tiles, hipStream_t st) {
    const size_t lds = p8_chunk_lds(DP, NQ, NS);
    auto fn = paged8_chunk_kernel<DP, NQ, NS, ONE>;
    static size_t done[16] = {};
    if (!reserve_lds(reinterpret_cast<const void*>(fn), lds, done))
        return fail(DKV_ELAUNCH, "dkv_paged8_attention: cannot reserve " + std::to_string(lds) + " B of LDS");
    hipLaunchKernelGGL(fn, dim3(a.c.n_kv_heads * a.c.batch, (int)((tiles + NQ - 1) / NQ), ONE ? 1 : p.slots + 1), dim3(512), lds, st, a);
    return DKV_OK;
}

template <int DP, int NS>
static int p8_launch(P8Args& a, const P8Plan& p, hipStream_t st) {
    const int64_t tiles = ((int64_t)a.T * (a.Hq / a.c.n_kv_heads) + 15) / 16;
    constexpr int NQ2 = DP <= 128 ? 2 : 1;   // (wider heads never have two)
    int rc;
    if (p.walk) rc = p8_launch_walk<DP, NS>(a, p, tiles, st);
    else if (p.nq == 1) rc = p.direct ? p8_launch_chunk<DP, 1, NS, true>(a, p, tiles, st) : p8_launch_chunk<DP, 1, NS, false>(a, p, tiles, st);
    else rc = p.direct ? p8_launch_chunk<DP, NQ2, NS, true>(a, p, tiles, st) : p8_launch_chunk<DP, NQ2, NS, false>(a, p, tiles, st);
    if (rc || (rc = check_launch("dkv_paged8_attention")) || p.direct) return rc;
    const int64_t rows = (int64_t)a.c.batch * a.T * a.Hq;
    hipLaunchKernelGGL((paged8_merge_kernel<DP, NS>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
    return check_launch("dkv_paged8_attention(merge)");
}

template <int NS>
static int p8_launch_ns(P8Args& a, const P8Plan& p, hipStream_t st) {
    switch (p8_dp(a.c.head_dim)) {
        case 32: return p8_launch<32, NS>(a, p, st);
        case 64: return p8_launch<64, NS>(a, p, st);
        case 128: return p8_launch<128, NS>(a, p, st);
        case 192: return p8_launch<192, NS>(a, p, st);
        default: return p8_launch<256, NS>(a, p, st);
    }
}

}  // namespace dkv

extern "C" size_t dkv_paged8_attention_workspace(const dkv_paged8_t* cache, int32_t T, int32_t n_q_heads,
                                                 int32_t max_len) {
    if (!cache || T <= 0 || n_q_heads <= 0 || max_len <= 0 || max_len > dkv::P8_MAX_LEN || cache->n_kv_heads <= 0 ||
        cache->head_dim <= 0 || cache->head_dim > dkv::P8_MAXD || cache->batch <= 0 || n_q_heads % cache->n_kv_heads)
        return 0;
    // (whichever type the queries have)
    return std::max(dkv::p8_plan(*cache, T, n_q_heads, max_len, 1).bytes, dkv::p8_plan(*cache, T, n_q_heads, max_len, 3).bytes);
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
    DKV_REQUIRE(max_len <= P8_MAX_LEN, "dkv_paged8_attention: max_len too large");
    if (T <= 0) return DKV_OK;
    if ((rc = p8_check_hot(c, T, "dkv_paged8_attention"))) return rc;
    const P8Plan p = p8_plan(c, T, n_q_heads, max_len, q_dtype == DKV_BF16 ? 1 : 3);
    DKV_REQUIRE((int64_t)c.batch * T * n_q_heads < (1LL << 31), "dkv_paged8_attention: too many rows");
    if (p.bytes && (!work || work_bytes < p.bytes || reinterpret_cast<uintptr_t>(work) % 16))
        return fail(DKV_EWORKSPACE, "dkv_paged8_attention: workspace too small or not 16-byte aligned (need " +
                                        std::to_string(p.bytes) + ")");
    P8Args a = {};
    a.c = c, a.layer = layer, a.T = T, a.Hq = n_q_heads;
    a.in_ring = p8_in_ring(c, T);
    a.bshift = __builtin_ctz(c.block_size);
    a.n_chunks = p.n_chunks, a.per_slot = p.per_slot, a.direct = p.direct;
    a.vec = c.head_dim % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    a.q = q, a.start = start, a.count = count, a.out = out;
    a.qscale = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(c.head_dim)));
    a.part = static_cast<float*>(work);
    a.ml = reinterpret_cast<float2*>(a.part + (int64_t)c.batch * T * n_q_heads * (p.n_chunks + 1) * p8_dp(c.head_dim));
    return q_dtype == DKV_BF16 ? p8_launch_ns<1>(a, p, as_stream(stream)) : p8_launch_ns<3>(a, p, as_stream(stream));
}
