// Causal attention over a paged full cache whose sequences share pages: the
// keys that the sequences of a group have in common are read once for all of
// them. Reference: the read + softmax of draftkv/llama.py:202-218 (there every
// sequence owns its rows).
//
//     s_k = q . K_k / sqrt(D),  out = sum_k 2^(s_k - m) V_k / sum_k 2^(s_k - m)
//     over the keys k <= position of the row (scores in base 2, m their maximum)
//
// Of a row's keys the first B, what its group shares rounded down to 32, are cut into pieces of `prefix` keys, the others
// from B on into units of `unit`. A row's state (m, l, o) over a piece is computed on its own by an online softmax in
// steps of 32 keys, and the merge adds a row's pieces in an order of their own. So a row's result is a function of its
// keys and B alone: not of T, nor of the other rows of the call. A piece of shared keys is computed for 32 rows of any of
// the group's sequences at a time, the others for 32 rows of one sequence.
//
// Products, the keys as the A operand:
//     S^T[32 keys][32 rows] = K . Q^T,   O^T[32 d][32 rows] += V^T . P^T
// Row m of the A operand of the first is key m with bits 2 and 3 exchanged: the
// accumulator then leaves a lane with keys 16 x + 8 (lane / 32) + 0 .. 7 of one
// row, which is what the B operand of the second takes, and V^T's operand is 16
// contiguous bytes. The probabilities never leave their lane.
//   bf16 cache, float32 queries: queries and probabilities in three bf16 parts
//     (24 bits, as much as float32 has) against the exact K and V
//   bf16 cache, bf16 queries: queries whole, probabilities in two parts (2^-16
//     of each, far below the rounding of the bf16 output)
//   float32 cache: float32 matrix instructions
//
// Two roles (measured at the choice, dkv_shared_attention()). Where a unit's
// rows are three tiles or more, the four waves of a workgroup take four tiles
// and share its keys through a ring of four stages in LDS: K and V come from
// L2 once for 128 rows. Otherwise each wave has a tile and a unit of its own and
// one stage: many short units are in flight, which is what hides their latency.
//
// Bound (32 / 8 heads of 128, bf16 cache; under the profiler):
//   many rows: the matrix cores. 32 sequences x 5 rows on 32.7k shared keys and
//     100 of their own, float32 queries: 230 us, 258 GFLOP in parts at 1120
//     TFLOP/s (a large library product 1164). One row each: 64 us; 256
//     workgroups walk the shared keys, one per CU, and 128 the others beside
//     them; 5 in the merge. Twice the workgroups with half the keys 62, and 7.
//   few rows: memory. 4 prompts of 16k x 16 sequences, bf16 queries: 83 us, 367
//     MB at 4.4 TB/s (a large copy 4.83).
//   small calls: the chain of loads before the first product and the steps of a
//     unit. 4 sequences on 500 rows, 9 / 3 heads of 64, float32: 11 us and 4 for
//     the merge.
#include <algorithm>
#include <type_traits>

#include "dkv_common.h"
#include "shared_plan.h"

// (every instantiation rounds alike, whatever the compiler would fuse in it)
#pragma clang fp contract(off)

namespace dkv {

typedef __bf16 sa_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 sa_bf16x2 __attribute__((ext_vector_type(2)));
typedef float sa_f32x2 __attribute__((ext_vector_type(2)));
typedef float sa_f32x4 __attribute__((ext_vector_type(4)));
typedef float sa_f32x16 __attribute__((ext_vector_type(16)));
// (callers' q and out need their elements' alignment only)
typedef float sa_f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t sa_u16x4u __attribute__((ext_vector_type(4), aligned(2)));

constexpr int SA_ROWS = 32, SA_WAVES = 4;
static_assert(SA_THREADS == 64 * SA_WAVES, "launches are cut by it");

struct SharedArgs {
    dkv_paged_t c;
    int layer, T, Hq, G;
    int t0, Tn;              // the rows of this launch: t0 .. t0 + Tn - 1 of every sequence
    int prefix, unit;        // keys per piece of what groups share, and per unit of what sequences have of their own
    int n_groups;
    int units_p, tiles_p;    // prefix tasks: pieces and row tiles per (group, KV head)
    int units_s, tiles_s;    // the sequences' own: units and row tiles per (sequence, KV head)
    int n_slots;             // a row's partials: units_p, then units_s
    bool wide_p, wide_s;     // a workgroup's waves share a unit's keys
    int64_t blocks_p, tasks_p, tasks_s;   // prefix workgroups; tasks of waves, or of (unit, head) pairs where wide
    const int32_t* first;    // [n_groups + 1]
    const int32_t* shared;   // [batch]
    const void* q;
    const int32_t* start;
    const int32_t* count;
    float qscale;            // log2(e) / sqrt(head_dim)
    float* part;             // o [row of the launch][n_slots][D]
    float2* ml;              // (m, l) [row of the launch][n_slots]
    void* out;
};

__device__ __forceinline__ float sa_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// the value of the other 32-lane half combined with the lane's own, the same bits in both
__device__ __forceinline__ float sa_max_halves(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sa_sum_halves(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// a, b as NS bf16 parts each, into elements k and k + 1
template <int NS>
__device__ __forceinline__ void sa_split(float a, float b, sa_bf16x8 (&o)[NS], int k) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const sa_bf16x2 h = __builtin_convertvector((sa_f32x2){a, b}, sa_bf16x2);
        o[i][k] = h[0], o[i][k + 1] = h[1];
        if (i + 1 < NS) {
            const uint32_t u = __builtin_bit_cast(uint32_t, h);
            a -= __uint_as_float(u << 16), b -= __uint_as_float(u & 0xffff0000u);
        }
    }
}

// at most N of the wave's loads still in flight; its LDS reads and writes done
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// the key of row m of a K operand: bits 2 and 3 exchanged
__device__ __forceinline__ int sa_key_of(int m) { return (m & 0x13) | (m & 4) << 1 | (m & 8) >> 1; }

// rows a sequence has after this call, within its block table
__device__ __forceinline__ int sa_len(const SharedArgs& A, int s) {
    return min(A.start[s] + (A.count ? A.count[s] : A.T), A.c.max_blocks * A.c.block_size);
}

// the keys that sequence s shares, as they are cut
__device__ __forceinline__ int sa_shared(const SharedArgs& A, int s) {
    return A.units_p ? min(min(max(A.shared[s], 0), A.c.max_blocks * A.c.block_size), A.units_p * A.prefix) & -SA_STEP : 0;
}
// the pieces of a row whose last key is `last`, `np` of them shared
__device__ __forceinline__ int sa_pieces(const SharedArgs& A, int last, int B, int& np) {
    if (last < 0) return np = 0;
    if (last < B) return np = last / A.prefix + 1;
    np = (B + A.prefix - 1) / A.prefix;
    return np + min((last - B) / A.unit + 1, A.units_s);
}

// Staging of the FAST path: 1 KB loads straight to LDS, 16 bytes per lane, into a step's 32 keys of K and V.
//   K: of 16 keys, 64 bytes each (channels 64 B * piece ..): lane = 16 * (16-byte chunk) + key. A K operand of the
//     product (16 bytes of channels of one key per lane) is one conflict-free 16-byte read.
//   V^T: rows of 16 keys as they lie in the page, but for a swap of 16-byte chunks between rows (sa_v_chunk), so that
//     an operand read covers all banks.
template <bool F32, int DP>
struct SharedStage {
    static constexpr int ESIZE = F32 ? 4 : 2;
    static constexpr int KPC = DP * ESIZE / 64;      // K loads per 16 keys
    static constexpr int K_BYTES = 2 * KPC * 1024;
    static constexpr int VROWS = 1024 / (16 * ESIZE);   // V^T rows per load
    static constexpr int VPC = DP / VROWS;           // V loads per 16 keys
    static constexpr int V_BYTES = 2 * VPC * 1024;
    static constexpr int LOADS = 2 * KPC + 2 * VPC;
    static constexpr int BYTES = K_BYTES + V_BYTES;
    static constexpr int STAGES = 4;                 // of a block's waves together; a wave alone has one of them
    static_assert(KPC == VPC && LOADS % SA_WAVES == 0, "loads split evenly");
};
// where the 16-byte chunk of a V^T row lies (its own inverse)
template <bool F32>
__device__ __forceinline__ int sa_v_chunk(int row, int chunk) {
    return F32 ? chunk ^ (row >> 2 & 3) : chunk ^ (row >> 3 & 1);
}

// A wave's task: a tile of 32 rows of one KV head and a unit of keys. The lane's row, and what is the same in the wave.
struct SharedTask {
    int slot, h, s0;         // the piece's partial, KV head, the sequence whose table is read
    int k_begin, k_there;    // the piece's first key, and where its keys that are there end
    int w_last, w_all;       // the last key that any row of the wave sees, and that all of them see
    bool rvalid, live;       // the lane has a row; it sees a key
    bool alone;              // and no piece but one
    int last, row_last;      // the row's last key; the same, and no bound for rows that do not count
    int64_t orow, prow;      // rows of q and out, and of the partials
};

// tile, u, h, s0: the same in the wave. False: no such task. k_begin is -1 where the sequence has no such unit.
__device__ __forceinline__ bool sa_task(const SharedArgs& A, bool prefix, int tile, int u, int h, int s0, int members, int B, SharedTask& k) {
    const dkv_paged_t& c = A.c;
    const int lane = threadIdx.x % WAVE, col = lane % 32;
    const int per = A.Tn * A.G, n_rows = members * per, r0 = tile * SA_ROWS;   // rows of one sequence, of all
    k.h = h, k.s0 = s0;
    k.slot = prefix ? u : A.units_p + u;
    const int len = __builtin_amdgcn_readfirstlane(sa_len(A, s0));
    k.k_begin = prefix ? u * A.prefix : sa_unit_begin(B, u, A.unit, len);
    k.rvalid = r0 + col < n_rows;
    const int r = min(r0 + col, n_rows - 1);
    const int s = s0 + r / per, t = A.t0 + r % per / A.G, hq = h * A.G + r % A.G;
    k.last = min(A.start[s] + t, sa_len(A, s) - 1);
    k.live = k.rvalid && k.last >= 0;
    k.orow = ((int64_t)s * A.T + t) * A.Hq + hq;
    k.prow = (((int64_t)s * A.Tn + (t - A.t0)) * A.Hq + hq) * A.n_slots;
    int np;
    k.alone = sa_pieces(A, k.last, B, np) <= 1 || A.n_slots == 1;
    int w_last = k.live ? k.last : -1, w_all = k.live ? k.last : INT_MAX;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        w_last = max(w_last, __shfl_xor(w_last, o));
        w_all = min(w_all, __shfl_xor(w_all, o));
    }
    k.w_last = __builtin_amdgcn_readfirstlane(w_last), k.w_all = __builtin_amdgcn_readfirstlane(w_all);
    k.row_last = k.live ? k.last : INT_MAX;
    k.k_there = prefix ? min(B, k.k_begin + A.prefix) : min(len, k.k_begin + A.unit);
    return r0 < n_rows;
}

// K and V^T operands: 16 (8) channels of a lane's key, 8 keys of a lane's channel; element by element from memory.
template <bool F32>
using sa_Kop = std::conditional_t<F32, sa_f32x4, sa_bf16x8>;
template <bool F32>
struct sa_Vop {
    sa_Kop<F32> v[F32 ? 2 : 1];
};
template <bool F32>
__device__ __forceinline__ sa_Kop<F32> sa_kop(const SharedArgs& A, const SharedTask& k, const int32_t* btab, int kb, int j) {
    constexpr int N = F32 ? 4 : 8;
    const dkv_paged_t& c = A.c;
    const int lane = threadIdx.x % WAVE, bs = c.block_size, kp = min(kb + sa_key_of(lane % 32), k.k_there - 1);
    const int32_t blk = btab[kp / bs];
    sa_Kop<F32> o;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int d = N * (2 * j + lane / 32) + e;
        const float x = d < c.head_dim ? load_elem(c.pool, paged_k_off(c, blk, kp % bs, k.h, d), c.dtype) : 0.0f;
        if constexpr (F32) o[e] = x;
        else o[e] = (__bf16)x;
    }
    return o;
}
// (past the cache's end zero: whatever the page holds, 0 * it could be NaN; FINITE: so are infinities and NaN)
template <bool F32, bool FINITE>
__device__ __forceinline__ sa_Vop<F32> sa_vop(const SharedArgs& A, const SharedTask& k, const int32_t* btab, int kb, int dt, int x) {
    const dkv_paged_t& c = A.c;
    const int lane = threadIdx.x % WAVE, bs = c.block_size, d = 32 * dt + lane % 32;
    sa_Vop<F32> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int vp = kb + 16 * x + 8 * (lane / 32) + e;
        float w = d < c.head_dim && vp < k.k_there ? load_elem(c.pool, paged_v_off(c, btab[vp / bs], vp % bs, k.h, d), c.dtype) : 0.0f;
        if (FINITE && !(fabsf(w) < INFINITY)) w = 0.0f;
        if constexpr (F32) v.v[e / 4][e % 4] = w;
        else v.v[0][e] = (__bf16)w;
    }
    return v;
}

// Scores to probabilities of a step's 16 keys of the lane, and the factor of what was summed before.
__device__ __forceinline__ float sa_softmax(const SharedArgs& A, const SharedTask& k, int kb, float (&p)[16], float& m_run, float& l_run) {
    if (kb + SA_STEP - 1 > k.w_all || kb + SA_STEP > k.k_there) {   // uniform: some row does not see the whole step
        const int lim = min(k.row_last, k.k_there - 1) - kb - 8 * (int)(threadIdx.x % WAVE / 32);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (16 * (i / 8) + i % 8 > lim) p[i] = -INFINITY;
    }
    float mx = p[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, p[i]);
    const float m_new = fmaxf(m_run, sa_max_halves(mx));
    const float ms = m_new == -INFINITY ? 0.0f : m_new;   // a row that sees no key yet: p = 0
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        p[i] = sa_exp2(p[i] - ms);
        sum += p[i];
    }
    const float alpha = m_new == m_run ? 1.0f : sa_exp2(m_run - m_new);
    l_run = l_run * alpha + sum;
    m_run = m_new;
    return alpha;
}

// One wave's walk: queries, sums and a step of 32 keys.
template <bool F32, bool QBF16, int DP>
struct SharedWalk {
    static constexpr int NS = QBF16 ? 1 : 3, PS = QBF16 ? 2 : 3;   // bf16 parts of queries and probabilities
    static constexpr int DT = DP / 32, KS = F32 ? DP / 8 : DP / 16;
    using Kop = sa_Kop<F32>;
    using Vop = sa_Vop<F32>;
    sa_bf16x8 qp[F32 ? 1 : KS][NS];
    sa_f32x4 qf[F32 ? KS : 1];
    sa_f32x16 acc[DT];
    float m_run, l_run;

    // channels 8 j + 4 half + e (float32 cache), 16 j + 8 half + e
    __device__ __forceinline__ void set_query(int j, const float* x, float qscale) {
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) qf[j][e] = x[e] * qscale;
        } else {
#pragma unroll
            for (int e = 0; e < 8; e += 2) {   // (bf16 queries stay whole: their scores are scaled)
                if constexpr (NS == 1) sa_split<NS>(x[e], x[e + 1], qp[j], e);
                else sa_split<NS>(x[e] * qscale, x[e + 1] * qscale, qp[j], e);
            }
        }
    }
    __device__ __forceinline__ void queries(const SharedArgs& A, const SharedTask& k) {   // any head_dim and alignment
        constexpr int N = F32 ? 4 : 8;
        const int half = threadIdx.x % WAVE / 32, D = A.c.head_dim;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            float x[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int d = N * (2 * j + half) + e;
                x[e] = d < D ? load_elem(A.q, k.orow * D + d, QBF16 ? DKV_BF16 : DKV_F32) : 0.0f;
            }
            set_query(j, x, A.qscale);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
        m_run = -INFINITY, l_run = 0.0f;
    }
    // Keys kb .. kb + 31. kop(j): the K operand of 16 (8) channels; between(): the scores are there, K is free; vop(dt, x):
    // the V^T operand of 32 channels and 16 keys. The lane holds key kb + 16 x + 8 half + e at 8 x + e.
    template <class K, class B, class V>
    __device__ __forceinline__ void step(const SharedArgs& A, const SharedTask& k, int kb, K&& kop, B&& between, V&& vop) {
        sa_f32x16 sc;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
            const Kop x = kop(j);
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], qf[j][e], sc, 0, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < NS; ++i) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, qp[j][i], sc, 0, 0, 0);
            }
        }
        between();
        float p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = !F32 && NS == 1 ? sc[i] * A.qscale : sc[i];
        const float alpha = sa_softmax(A, k, kb, p, m_run, l_run);
        if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][e] *= alpha;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            sa_bf16x8 pp[F32 ? 1 : PS];
            if constexpr (!F32)
#pragma unroll
                for (int e = 0; e < 8; e += 2) sa_split<PS>(p[8 * x + e], p[8 * x + e + 1], pp, e);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const Vop v = vop(dt, x);
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(v.v[e / 4][e % 4], p[8 * x + e], acc[dt], 0, 0, 0);
                } else {
#pragma unroll
                    for (int i = 0; i < PS; ++i)
                        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v.v[0], pp[i], acc[dt], 0, 0, 0);
                }
            }
        }
    }
    // The whole unit with K and V element by element from memory.
    __device__ __forceinline__ void unit(const SharedArgs& A, const SharedTask& k) {
        const int32_t* btab = A.c.block_table + ((int64_t)k.s0 * A.c.n_layers + A.layer) * A.c.max_blocks;
        clear();
        const int k_end = min(k.k_there, k.w_last + 1);
#pragma unroll 1
        for (int kb = k.k_begin; kb < k_end; kb += SA_STEP)
            step(A, k, kb, [&](int j) { return sa_kop<F32>(A, k, btab, kb, j); }, [] {},
                 [&](int dt, int x) { return sa_vop<F32, false>(A, k, btab, kb, dt, x); });
    }
    // The walk met a NaN: of a key that its row sees, or 0 times one that it does not.
    __device__ __forceinline__ bool odd() const {
        bool o = l_run != l_run;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o |= acc[dt][i] != acc[dt][i];
        return __builtin_amdgcn_readfirstlane(__any(o)) != 0;
    }
    __device__ __forceinline__ static void put(const SharedArgs& A, int64_t i, float x) {
        if constexpr (QBF16) static_cast<uint16_t*>(A.out)[i] = f32_to_bf16_rne(x);
        else static_cast<float*>(A.out)[i] = x;
    }
    // The row's state out: channels 32 dt + 8 (i / 4) + 4 half + i % 4. WIDE: head_dim is DP.
    template <bool WIDE>
    __device__ __forceinline__ void store(const SharedArgs& A, const SharedTask& k) const {
        const int half = threadIdx.x % WAVE / 32, D = WIDE ? DP : A.c.head_dim;
        const float l = sa_sum_halves(l_run);
        if (!k.live) return;
        const bool alone = k.alone;
        if (alone && k.k_begin > k.last) return;
        float* part = A.part + (k.prow + k.slot) * D;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = 32 * dt + 2 * i + 4 * half;
                if constexpr (WIDE) {
                    const sa_f32x4 o = {acc[dt][i], acc[dt][i + 1], acc[dt][i + 2], acc[dt][i + 3]};
                    if (!alone) {
                        *reinterpret_cast<sa_f32x4*>(part + d) = o;
                    } else if constexpr (QBF16) {
                        sa_u16x4u w;
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = f32_to_bf16_rne(o[e] / l);
                        *reinterpret_cast<sa_u16x4u*>(static_cast<uint16_t*>(A.out) + k.orow * D + d) = w;
                    } else {
                        *reinterpret_cast<sa_f32x4u*>(static_cast<float*>(A.out) + k.orow * D + d) = sa_f32x4u{o[0] / l, o[1] / l, o[2] / l, o[3] / l};
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (d + e >= D) continue;
                        if (alone) put(A, k.orow * D + d + e, acc[dt][i + e] / l);
                        else part[d + e] = acc[dt][i + e];
                    }
                }
            }
        if (!alone && half == 0) A.ml[k.prow + k.slot] = make_float2(m_run, l);
    }
};

// The unit again, for walks that met a NaN: of a key that its row sees, or 0 times what it does not. Infinities and NaN of
// V stay out of the products and go to the rows that see them by hand; other rows get the same bits. 32 channels at a time:
// it is rare, and must not be what the kernel's registers are counted by.
template <bool F32, bool QBF16>
__device__ __forceinline__ void sa_again(const SharedArgs& A, const SharedTask& k) {
    constexpr int NS = QBF16 ? 1 : 3, PS = QBF16 ? 2 : 3, N = F32 ? 4 : 8;
    const dkv_paged_t& c = A.c;
    const int lane = threadIdx.x % WAVE, col = lane % 32, half = lane / 32, D = c.head_dim, bs = c.block_size;
    const int32_t* btab = c.block_table + ((int64_t)k.s0 * c.n_layers + A.layer) * c.max_blocks;
    const int k_end = min(k.k_there, k.w_last + 1);
    auto q = [&](int d) { return d < D ? load_elem(A.q, k.orow * D + d, QBF16 ? DKV_BF16 : DKV_F32) : 0.0f; };
#pragma unroll 1
    for (int dt = 0; 32 * dt < D; ++dt) {
        sa_f32x16 acc;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
        float m_run = -INFINITY, l_run = 0.0f;
#pragma unroll 1
        for (int kb = k.k_begin; kb < k_end; kb += SA_STEP) {
            sa_f32x16 sc;
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
#pragma unroll 1
            for (int j = 0; 2 * N * j < (D + 31) / 32 * 32; ++j) {
                const sa_Kop<F32> x = sa_kop<F32>(A, k, btab, kb, j);
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], q(N * (2 * j + half) + e) * A.qscale, sc, 0, 0, 0);
                } else {
                    sa_bf16x8 qp[NS];
                    const float f = NS == 1 ? 1.0f : A.qscale;
#pragma unroll
                    for (int e = 0; e < 8; e += 2) sa_split<NS>(q(N * (2 * j + half) + e) * f, q(N * (2 * j + half) + e + 1) * f, qp, e);
#pragma unroll
                    for (int i = 0; i < NS; ++i) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, qp[i], sc, 0, 0, 0);
                }
            }
            float p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = !F32 && NS == 1 ? sc[i] * A.qscale : sc[i];
            if constexpr (!F32 && NS > 1) {
                // An infinity times a query's parts is no number where they differ in sign or one is 0: its score again,
                // channel by channel
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    __builtin_amdgcn_sched_barrier(0);
                    if (p[i] == p[i]) continue;
                    const int kp = min(kb + 16 * (i / 8) + 8 * half + i % 8, k.k_there - 1);
                    const int32_t blk = btab[kp / bs];
                    float x = 0.0f;
#pragma unroll 1
                    for (int d = 0; d < D; ++d) x += q(d) * A.qscale * load_elem(c.pool, paged_k_off(c, blk, kp % bs, k.h, d), c.dtype);
                    p[i] = x;
                }
            }
            const float alpha = sa_softmax(A, k, kb, p, m_run, l_run);
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] *= alpha;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                __builtin_amdgcn_sched_barrier(0);
                const sa_Vop<F32> v = sa_vop<F32, true>(A, k, btab, kb, dt, x);
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(v.v[e / 4][e % 4], p[8 * x + e], acc, 0, 0, 0);
                } else {
                    sa_bf16x8 pp[PS];
#pragma unroll
                    for (int e = 0; e < 8; e += 2) sa_split<PS>(p[8 * x + e], p[8 * x + e + 1], pp, e);
#pragma unroll
                    for (int i = 0; i < PS; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v.v[0], pp[i], acc, 0, 0, 0);
                }
            }
#pragma unroll 1
            for (int key = 0; key < SA_STEP && kb + key < k.k_there; ++key) {
                float pk = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) pk = 16 * (i / 8) + i % 8 == (key & ~8) ? p[i] : pk;
                pk = __shfl(pk, col + 4 * (key & 8));
                if (kb + key > k.row_last) continue;
                const int32_t blk = btab[(kb + key) / bs];
#pragma unroll
                for (int i = 0; i < 16; ++i) {   // the lane's channels
                    if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);
                    const int d = 32 * dt + 8 * (i / 4) + 4 * half + i % 4;
                    const float z = d < D ? load_elem(c.pool, paged_v_off(c, blk, (kb + key) % bs, k.h, d), c.dtype) : 0.0f;
                    if (!(fabsf(z) < INFINITY)) acc[i] += pk * z;
                }
            }
        }
        const float l = sa_sum_halves(l_run);
        if (!k.live || (k.alone && k.k_begin > k.last)) continue;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);
            const int d = 32 * dt + 8 * (i / 4) + 4 * half + i % 4;
            if (d >= D) continue;
            if (!k.alone) A.part[(k.prow + k.slot) * D + d] = acc[i];
            else if constexpr (QBF16) static_cast<uint16_t*>(A.out)[k.orow * D + d] = f32_to_bf16_rne(acc[i] / l);
            else static_cast<float*>(A.out)[k.orow * D + d] = acc[i] / l;
        }
        if (!k.alone && half == 0) A.ml[k.prow + k.slot] = make_float2(m_run, l);
    }
}

// DP: head_dim rounded up to 32. FAST: head_dim a multiple of 32, blocks of whole 16-token runs, an aligned pool.
template <bool F32, bool QBF16, int DP, bool FAST>
__global__ void __launch_bounds__(64 * SA_WAVES, 2) shared_attn_kernel(SharedArgs A) {
    using St = SharedStage<F32, DP>;
    using Walk = SharedWalk<F32, QBF16, DP>;
    using Kop = typename Walk::Kop;
    using Vop = typename Walk::Vop;
    const dkv_paged_t& c = A.c;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int col = lane % 32, half = lane / 32;
    const int bs = c.block_size, H = c.n_kv_heads;

    // ---- the wave's task, or, where there are many rows (wide), four tiles and a unit for the workgroup
    int64_t task = blockIdx.x;
    const bool prefix = task < A.blocks_p;
    const bool wide = FAST && (prefix ? A.wide_p : A.wide_s);
    const int tiles = prefix ? A.tiles_p : A.tiles_s, units = prefix ? A.units_p : A.units_s;
    if (!prefix) task -= A.blocks_p;
    int tile;
    if (wide) {
        // workgroups of one unit and head on one XCD (they are dealt out round robin): its L2 holds the keys
        const int tb = (tiles + SA_WAVES - 1) / SA_WAVES;
        const int64_t q = task / (8 * tb), r = task % (8 * tb);
        tile = (int)(r / 8) * SA_WAVES + wave;
        task = q * 8 + r % 8;
        if (task >= (prefix ? A.tasks_p : A.tasks_s)) return;
    } else {
        task = task * SA_WAVES + wave;
        if (task >= (prefix ? A.tasks_p : A.tasks_s)) return;
        tile = (int)(task % tiles), task /= tiles;
    }
    const int u = (int)(task % units);
    task /= units;
    const int h = (int)(task % H);
    int s0 = (int)(task / H), members = 1;
    if (prefix) {
        const int g = s0;
        s0 = __builtin_amdgcn_readfirstlane(min(max(A.first[g], 0), c.batch));
        members = __builtin_amdgcn_readfirstlane(min(max(A.first[g + 1], s0), c.batch)) - s0;
    }
    if (members <= 0) return;
    const int B = __builtin_amdgcn_readfirstlane(sa_shared(A, s0));
    if (prefix && u * A.prefix >= B) return;
    SharedTask k;
    const bool mine = sa_task(A, prefix, tile, u, h, s0, members, B, k);
    if (k.k_begin < 0) return;
    if (!mine && (!wide || (tile - wave) * SA_ROWS >= members * A.Tn * A.G)) return;
    if (k.k_begin == 0 && k.rvalid && !k.live)   // an empty sequence
        for (int d = half; d < c.head_dim; d += 2) Walk::put(A, k.orow * c.head_dim + d, 0.0f);
    if (!wide && k.w_last < k.k_begin) return;

    Walk w;
    if constexpr (!FAST) {
        w.queries(A, k);
        w.unit(A, k);
    } else {
        {   // whole vectors; loaded before any is used
            constexpr int N = F32 ? 4 : 8;
            float x[Walk::KS][N];
#pragma unroll
            for (int j = 0; j < Walk::KS; ++j)
#pragma unroll
                for (int y = 0; y < N; y += 4) {
                    const int64_t at = k.orow * DP + N * (2 * j + half) + y;
                    if constexpr (QBF16) {
                        const sa_u16x4u q = *reinterpret_cast<const sa_u16x4u*>(static_cast<const uint16_t*>(A.q) + at);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[j][y + e] = bf16_to_f32(q[e]);
                    } else {
                        const sa_f32x4u q = *reinterpret_cast<const sa_f32x4u*>(static_cast<const float*>(A.q) + at);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[j][y + e] = q[e];
                    }
                }
#pragma unroll
            for (int j = 0; j < Walk::KS; ++j) w.set_query(j, x[j], A.qscale);
        }
        // ---- K and V through LDS
        extern __shared__ __align__(16) char lds[];
        int k_last = k.w_last;   // the last key of any row that the stages are for
        if (wide) {
            int* wl = reinterpret_cast<int*>(lds);
            if (lane == 0) wl[wave] = k.w_last;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < SA_WAVES; ++i) k_last = max(k_last, wl[i]);
            k_last = __builtin_amdgcn_readfirstlane(k_last);
            __syncthreads();
            if (k_last < k.k_begin) return;
        }
        const int nsteps = (min(k.k_there, k_last + 1) - k.k_begin + SA_STEP - 1) / SA_STEP;
        const int32_t* btab = c.block_table + ((int64_t)s0 * c.n_layers + A.layer) * c.max_blocks;
        constexpr int ES = St::ESIZE;
        const int64_t block_bytes = paged_block_elems(c) * ES;
        // Where the 16-key runs from run0 on begin, one per lane (the last run that is there for those past it): byte
        // offsets of the head's rows of K and of V^T in the pool. Worked out here once for 64 runs: in scalar registers at
        // each load it was 140 instructions a step, as long as the step's products.
        const int last_run = (k.k_there - 1) / 16, first_run = k.k_begin / 16;
        int run0 = first_run;
        int64_t at_k, at_v;
        auto load_ids = [&]() {
            const int pos = min(run0 + lane, last_run) * 16;
            const int64_t block = btab[pos / bs] * block_bytes;
            at_k = block + ((int64_t)h * bs + pos % bs) * DP * ES;
            at_v = block + (((int64_t)H + h) * bs * DP + pos % bs) * ES;
        };
        load_ids();
        auto base = [&](int64_t at, int run) -> const char* {   // run: uniform
            const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)at, run - run0);
            const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)at >> 32), run - run0);
            return static_cast<const char*>(c.pool) + (int64_t)((uint64_t)hi << 32 | lo);
        };
        // byte offsets of the lane in a load: K rows, V^T rows
        const uint32_t klane = (uint32_t)((lane % 16) * DP * ES + lane / 16 * 16);
        constexpr int VL = ES;   // 16-byte chunks of a V^T row of 16 keys
        // (the swap is the same in every load: their rows are 16 or 32 apart)
        const uint32_t vlane = (uint32_t)(lane / VL * bs * ES + sa_v_chunk<F32>(lane / VL, lane % VL) * 16);
        const int64_t vpiece = (int64_t)St::VROWS * bs * ES;
        const uint32_t kread = (uint32_t)((sa_key_of(col) >> 4) * St::KPC * 1024 + half * 256 + (sa_key_of(col) & 15) * 16);
        auto kop_at = [&](const char* st, int j) {
            return *reinterpret_cast<const Kop*>(st + kread + (j >> 1) * 1024 + (j & 1) * 512);
        };
        auto vop_at = [&](const char* st, int dt, int x) {
            Vop v;
#pragma unroll
            for (int y = 0; y < (F32 ? 2 : 1); ++y) {
                const int chunk = sa_v_chunk<F32>(col, F32 ? 2 * half + y : half);
                v.v[y] = *reinterpret_cast<const Kop*>(st + St::K_BYTES + (x * DP + 32 * dt + col) * (16 * ES) + chunk * 16);
            }
            return v;
        };
        // V^T past the cache's end becomes zero
        auto zero_past = [&](char* st, int live_keys, int thread, int threads) {
            for (int i = thread; i < St::V_BYTES / 16; i += threads) {
                const int row = i / VL % DP, key = 16 * (i / VL / DP) + sa_v_chunk<F32>(row, i % VL) * (16 / ES);
#pragma unroll
                for (int e = 0; e < 16 / ES; ++e)
                    if (key + e >= live_keys) {
                        if constexpr (F32) reinterpret_cast<float*>(st + St::K_BYTES + 16 * i)[e] = 0.0f;
                        else reinterpret_cast<uint16_t*>(st + St::K_BYTES + 16 * i)[e] = 0;
                    }
            }
        };
        w.clear();
        if (wide) {
            constexpr int S = St::STAGES, LPW = St::LOADS / SA_WAVES;
            // this wave's share of step i's loads: K or V of one of its two runs
            const bool is_v = wave >= 2;
            const int64_t piece = is_v ? vpiece : 64;
            const uint32_t off = is_v ? vlane : klane;
            auto issue = [&](int i) {
                const char* from = base(is_v ? at_v : at_k, first_run + 2 * i + (wave & 1));
                const uint32_t to = lds_offset(lds) + (i % S) * St::BYTES + wave * LPW * 1024;
#pragma unroll
                for (int x = 0; x < LPW; ++x) dma_b128<false>(from + x * piece, off, to + x * 1024);
            };
            static_assert(LPW == St::KPC && SA_WAVES == 4, "a wave loads K or V of one run");
#pragma unroll
            for (int i = 0; i < S - 1; ++i)
                if (i < nsteps) issue(i);
            for (int i = 0; i < nsteps; ++i) {
                // this wave's loads of step i are done once those of the S - 2 later steps alone remain; the barrier
                // makes every wave's visible, and frees the stage of step i - 1
                const int later = min(S - 2, nsteps - 1 - i);
                if (later >= 2) wait_loads_barrier<2 * LPW>();
                else if (later == 1) wait_loads_barrier<LPW>();
                else wait_loads_barrier<0>();
                if (i + S - 1 < nsteps) {
                    if (first_run + 2 * (i + S - 1) - run0 >= WAVE) run0 += WAVE, load_ids();
                    issue(i + S - 1);
                }
                const int kb = k.k_begin + SA_STEP * i;
                char* st = lds + (i % S) * St::BYTES;
                if (kb + SA_STEP > k.k_there) {
                    zero_past(st, k.k_there - kb, threadIdx.x, 64 * SA_WAVES);
                    __syncthreads();
                }
                if (kb > k.w_last) continue;   // uniform over the wave
                w.step(A, k, kb, [&](int j) { return kop_at(st, j); }, [] {}, [&](int dt, int x) { return vop_at(st, dt, x); });
            }
        } else {
            // one stage: K of the next step is fetched once this one's scores are there, V once its products are
            char* st = lds + wave * St::BYTES;
            const uint32_t to = lds_offset(st);
            auto issue_k = [&](int i) {
                const int run = first_run + 2 * i;
                if (run - run0 >= WAVE) run0 += WAVE, load_ids();
                const char* from[2] = {base(at_k, run), base(at_k, run + 1)};
#pragma unroll
                for (int x = 0; x < 2 * St::KPC; ++x) dma_b128<false>(from[x / St::KPC] + 64 * (x % St::KPC), klane, to + x * 1024);
            };
            auto issue_v = [&](int i) {   // (after its K: the offsets are there)
                const int run = first_run + 2 * i;
                const char* from[2] = {base(at_v, run), base(at_v, run + 1)};
#pragma unroll
                for (int x = 0; x < 2 * St::VPC; ++x)
                    dma_b128<false>(from[x / St::VPC] + (x % St::VPC) * vpiece, vlane, to + St::K_BYTES + x * 1024);
            };
            issue_k(0);
            issue_v(0);
            for (int i = 0; i < nsteps; ++i) {
                const int kb = k.k_begin + SA_STEP * i;
                const bool more = i + 1 < nsteps;
                wait_loads<2 * St::VPC>();   // K is there, V may be on its way
                w.step(A, k, kb, [&](int j) { return kop_at(st, j); },
                       [&]() {
                           wait_lds();
                           if (more) {
                               issue_k(i + 1);
                               wait_loads<2 * St::KPC>();
                           } else {
                               wait_loads<0>();
                           }
                           if (kb + SA_STEP > k.k_there) {
                               zero_past(st, k.k_there - kb, lane, WAVE);
                               wait_lds();
                           }
                       },
                       [&](int dt, int x) { return vop_at(st, dt, x); });
                if (more) {
                    wait_lds();
                    issue_v(i + 1);
                }
            }
        }
        if (!mine || k.w_last < k.k_begin) return;
    }
    if (!w.odd()) {
        w.template store<FAST>(A, k);
        return;
    }
    sa_again<F32, QBF16>(A, k);
}

// Merge of each row's pieces: their common maximum first, then the weighted
// sums, pieces u, u + 4, ... in order and these four last, so the result depends
// on the row's pieces alone. Four waves per row, one class each; a lane weighs
// the piece of its number and holds channels 2 lane and 2 lane + 1. Eight
// pieces' loads are in flight at once, the first beside the weights'. Bound: a
// chain of three loads where rows are few (4 us), else memory: 5120 rows of 32
// pieces and one, 88 MB in 18 us.
constexpr int SM_CLASSES = 4;
static_assert(SA_THREADS == 64 * SM_CLASSES, "launches are cut by it");
template <bool QBF16>
__global__ void __launch_bounds__(64 * SM_CLASSES) shared_merge_kernel(SharedArgs A) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE, D = A.c.head_dim;
    int64_t i = blockIdx.x;
    const int hq = (int)(i % A.Hq);
    i /= A.Hq;
    const int t = A.t0 + (int)(i % A.Tn), s = (int)(i / A.Tn);
    const int last = min(A.start[s] + t, sa_len(A, s) - 1);
    int np;
    const int n = __builtin_amdgcn_readfirstlane(sa_pieces(A, last, sa_shared(A, s), np));
    if (n <= 1) return;   // the attention kernel wrote the row
    np = __builtin_amdgcn_readfirstlane(np);
    const int64_t prow = (int64_t)blockIdx.x * A.n_slots;
    auto slot = [&](int i) { return prow + (i < np ? i : A.units_p + i - np); };
    const int c0 = min(2 * lane, D - 1), c1 = min(2 * lane + 1, D - 1);
    const bool pair = D % 2 == 0;
    float2 v[8];
    auto fetch = [&](int u0, int u, int ue) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float* p = A.part + slot(u0 + min(u + k * SM_CLASSES, ue - 1)) * D;
            v[k] = pair ? *reinterpret_cast<const float2*>(p + min(c0, D - 2)) : make_float2(p[c0], p[c1]);
        }
    };
    // the first loads at once: the lanes' weights and the class's first eight pieces
    const float2 x0 = A.ml[slot(min(lane, n - 1))];
    fetch(0, w, min(n, WAVE));
    float m = x0.x;
    for (int u = lane + WAVE; u < n; u += WAVE) m = fmaxf(m, A.ml[slot(u)].x);
    m = wave_max(m);
    const float ms = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int u0 = 0; u0 < n; u0 += WAVE) {
        float f = 0.0f;
        if (u0 + lane < n) {
            float2 x = x0;
            if (u0 > 0) x = A.ml[slot(u0 + lane)];
            f = sa_exp2(x.x - ms);
            l = fmaf(x.y, f, l);
        }
        const int ue = min(n - u0, WAVE);
        for (int u = w; u < ue; u += 8 * SM_CLASSES) {
            if (u0 > 0 || u > w) fetch(u0, u, ue);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (u + k * SM_CLASSES < ue) {
                    const float g = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(f), u + k * SM_CLASSES));
                    o0 = fmaf(v[k].x, g, o0);
                    o1 = fmaf(v[k].y, g, o1);
                }
        }
    }
    __shared__ float2 so[SM_CLASSES][WAVE];
    if (w > 0) so[w][lane] = make_float2(o0, o1);
    __syncthreads();
    if (w > 0) return;
    const float lt = wave_sum(l);   // (every wave holds all of l)
    if (2 * lane >= D) return;
#pragma unroll
    for (int k = 1; k < SM_CLASSES; ++k) o0 += so[k][lane].x, o1 += so[k][lane].y;
    const int64_t at = (((int64_t)s * A.T + t) * A.Hq + hq) * D + 2 * lane;
    if constexpr (QBF16) {
        static_cast<uint16_t*>(A.out)[at] = f32_to_bf16_rne(o0 / lt);
        if (2 * lane + 1 < D) static_cast<uint16_t*>(A.out)[at + 1] = f32_to_bf16_rne(o1 / lt);
    } else {
        static_cast<float*>(A.out)[at] = o0 / lt;
        if (2 * lane + 1 < D) static_cast<float*>(A.out)[at + 1] = o1 / lt;
    }
}

// Rows per launch: as many of the T as keep the partials within this, and the merge's workgroups within a launch
constexpr size_t SA_WORK_BYTES = (size_t)512 << 20;
static size_t sa_row_bytes(const dkv_paged_t& c, int Hq, int n_slots) {   // of one t
    return sizeof(float) * (size_t)c.batch * Hq * n_slots * (c.head_dim + 2);
}
static int sa_rows(const dkv_paged_t& c, int T, int Hq, int n_slots) {
    const size_t most = std::min<size_t>(SA_WORK_BYTES / sa_row_bytes(c, Hq, n_slots), SA_BLOCKS / ((int64_t)c.batch * Hq));
    return (int)std::min<size_t>(T, std::max<size_t>(1, most));
}
static void sa_units(const dkv_paged_t& c, const dkv_groups_t& g, int max_len, int prefix, int unit, int& units_p, int& units_s) {
    sa_units((int64_t)c.max_blocks * c.block_size, max_len, g.n_groups > 0, g.min_shared, g.max_shared, prefix, unit, units_p, units_s);
}

template <bool F32, bool QBF16, int DP, bool FAST>
static int sa_launch_one(const SharedArgs& a, dim3 grid, hipStream_t st) {
    auto kfn = shared_attn_kernel<F32, QBF16, DP, FAST>;
    const size_t lds = FAST ? SharedStage<F32, DP>::BYTES * SharedStage<F32, DP>::STAGES : 0;
    static size_t lds_done[16] = {};
    if (!reserve_lds(reinterpret_cast<const void*>(kfn), lds, lds_done))
        return fail(DKV_ELAUNCH, "dkv_shared_attention: cannot reserve " + std::to_string(lds) + " B of LDS");
    hipLaunchKernelGGL(kfn, grid, dim3(64 * SA_WAVES), lds, st, a);
    return check_launch("dkv_shared_attention");
}
template <bool F32, bool QBF16, bool FAST>
static int sa_launch(const SharedArgs& a, dim3 grid, hipStream_t st) {
    switch ((a.c.head_dim + 31) / 32) {
        case 1: return sa_launch_one<F32, QBF16, 32, FAST>(a, grid, st);
        case 2: return sa_launch_one<F32, QBF16, 64, FAST>(a, grid, st);
        case 3: return sa_launch_one<F32, QBF16, 96, FAST>(a, grid, st);
        default: return sa_launch_one<F32, QBF16, 128, FAST>(a, grid, st);
    }
}

static int sa_check(const dkv_paged_t& c, const dkv_groups_t& g, int T, int Hq, int max_len, int prefix, int unit) {
    DKV_REQUIRE(c.dtype == DKV_F32 || c.dtype == DKV_BF16, "dkv_shared_attention: bad cache dtype");
    DKV_REQUIRE(c.batch > 0 && c.n_layers > 0 && c.n_kv_heads > 0 && c.block_size > 0 && c.max_blocks > 0,
                "dkv_shared_attention: bad cache shape");
    DKV_REQUIRE((int64_t)c.max_blocks * c.block_size < (1LL << 31) - SA_MOST_KEYS, "dkv_shared_attention: more than 2^31 positions");
    DKV_REQUIRE(c.head_dim > 0 && c.head_dim <= 128, "dkv_shared_attention: head_dim must be 1..128");
    DKV_REQUIRE(Hq > 0 && Hq % c.n_kv_heads == 0, "dkv_shared_attention: query heads must be a multiple of KV heads");
    DKV_REQUIRE(unit > 0 && unit <= SA_MOST_KEYS && unit % SA_STEP == 0,
                "dkv_shared_attention: unit_keys must be a multiple of 32, at most 65536");
    DKV_REQUIRE(prefix > 0 && prefix <= SA_MOST_KEYS && prefix % SA_STEP == 0,
                "dkv_shared_attention: prefix_keys must be a multiple of 32, at most 65536");
    DKV_REQUIRE(max_len > 0, "dkv_shared_attention: max_len must be > 0");
    DKV_REQUIRE(T >= 0 && (int64_t)c.batch * T * Hq < (1LL << 31), "dkv_shared_attention: too many rows");
    // (a padding row's position is formed before it is cut to the last one's)
    DKV_REQUIRE((int64_t)c.max_blocks * c.block_size + T < (1LL << 31), "dkv_shared_attention: positions past 2^31 (the table's, and T more)");
    DKV_REQUIRE(g.n_groups >= 0 && g.n_groups <= c.batch, "dkv_shared_attention: n_groups must lie in 0..batch");
    DKV_REQUIRE(g.n_groups == 0 || (g.max_members > 0 && g.max_members <= c.batch && g.min_shared >= 0 &&
                                    g.min_shared <= g.max_shared),
                "dkv_shared_attention: bad group bounds");
    return DKV_OK;
}

}  // namespace dkv

extern "C" size_t dkv_shared_attention_workspace(const dkv_paged_t* cache, const dkv_groups_t* groups, int32_t T,
                                                 int32_t n_q_heads, int32_t max_len, int32_t prefix_keys, int32_t unit_keys) {
    if (!cache || !groups || T <= 0 || dkv::sa_check(*cache, *groups, T, n_q_heads, max_len, prefix_keys, unit_keys)) return 0;
    int p, s;
    dkv::sa_units(*cache, *groups, max_len, prefix_keys, unit_keys, p, s);
    if (p + s <= 1) return 0;
    return dkv::sa_rows(*cache, T, n_q_heads, p + s) * dkv::sa_row_bytes(*cache, n_q_heads, p + s) + 8;   // (m, l) on 8 bytes
}

extern "C" int dkv_shared_attention(const dkv_paged_t* cache, const dkv_groups_t* groups, int32_t layer, const void* q,
                                    int32_t q_dtype, int32_t T, int32_t n_q_heads, const int32_t* start,
                                    const int32_t* count, int32_t max_len, int32_t prefix_keys, int32_t unit_keys, void* out,
                                    void* work, size_t work_bytes, dkv_stream_t stream) {
    using namespace dkv;
    DKV_REQUIRE(cache && groups, "dkv_shared_attention: NULL argument");
    const dkv_paged_t c = *cache;
    const dkv_groups_t g = *groups;
    const int rc = sa_check(c, g, T, n_q_heads, max_len, prefix_keys, unit_keys);
    if (rc) return rc;
    DKV_REQUIRE(layer >= 0 && layer < c.n_layers, "dkv_shared_attention: layer out of range");
    DKV_REQUIRE(q_dtype == DKV_F32 || q_dtype == DKV_BF16, "dkv_shared_attention: bad query dtype");
    if (T == 0) return DKV_OK;
    DKV_REQUIRE(q && start && out && c.pool && c.block_table && (g.n_groups == 0 || (g.first && g.shared)),
                "dkv_shared_attention: NULL argument");
    SharedArgs a = {};
    a.c = c, a.layer = layer, a.T = T, a.Hq = n_q_heads, a.G = n_q_heads / c.n_kv_heads;
    a.prefix = prefix_keys, a.unit = unit_keys;
    sa_units(c, g, max_len, prefix_keys, unit_keys, a.units_p, a.units_s);
    a.n_slots = a.units_p + a.units_s;
    a.n_groups = g.n_groups, a.first = g.first, a.shared = g.shared;
    a.q = q, a.start = start, a.count = count, a.out = out;
    a.qscale = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(c.head_dim)));
    const size_t need = dkv_shared_attention_workspace(cache, groups, T, n_q_heads, max_len, prefix_keys, unit_keys);
    if (need && (!work || work_bytes < need))
        return fail(DKV_EWORKSPACE, "dkv_shared_attention: workspace too small (need " + std::to_string(need) + ")");
    const int step = sa_rows(c, T, n_q_heads, a.n_slots);
    hipStream_t st = as_stream(stream);
    const bool f32 = c.dtype == DKV_F32, qb = q_dtype == DKV_BF16;
    // (by whole vectors through LDS, or element by element: 32 sequences on 16k 47 us and 527, 4 on 500 float32 17 and 39)
    const bool fast = c.block_size % 16 == 0 && c.head_dim % 32 == 0 && reinterpret_cast<uintptr_t>(c.pool) % 16 == 0;
    for (a.t0 = 0; a.t0 < T; a.t0 += step) {
        a.Tn = std::min(step, T - a.t0);
        const int64_t rows = (int64_t)c.batch * a.Tn * n_q_heads;
        a.part = static_cast<float*>(work);
        a.ml = reinterpret_cast<float2*>(a.part + (rows * a.n_slots * c.head_dim + 1) / 2 * 2);
        const int64_t per = (int64_t)a.Tn * a.G;
        a.tiles_p = (int)((g.max_members * per + SA_ROWS - 1) / SA_ROWS);
        a.tiles_s = (int)((per + SA_ROWS - 1) / SA_ROWS);
        // (unit, head) pairs; a workgroup's four waves take four tiles of one (wide), or four tasks of a tile each
        const int64_t pairs_p = (int64_t)a.n_groups * c.n_kv_heads * a.units_p, pairs_s = (int64_t)c.batch * c.n_kv_heads * a.units_s;
        // (us, wide and not; one row each on 16k shared keys, 32 / 8 heads of 128, bf16 cache: four groups of 8, 16, 24 and 32
        // sequences, 1, 2, 3 and 4 tiles: 88 / 59, 112 / 84, 118 / 131, 134 / 142; 20 tiles on 32k 257 / 298)
        a.wide_p = fast && a.tiles_p >= 3, a.wide_s = fast && a.tiles_s >= 3;
        auto blocks_of = [](bool wide, int64_t pairs, int tiles, int64_t& tasks) {
            tasks = wide ? pairs : pairs * tiles;
            return wide ? (pairs + 7) / 8 * 8 * ((tiles + SA_WAVES - 1) / SA_WAVES) : (tasks + SA_WAVES - 1) / SA_WAVES;
        };
        a.blocks_p = blocks_of(a.wide_p, pairs_p, a.tiles_p, a.tasks_p);
        const int64_t blocks = a.blocks_p + blocks_of(a.wide_s, pairs_s, a.tiles_s, a.tasks_s);
        DKV_REQUIRE(blocks <= SA_BLOCKS && (a.n_slots == 1 || rows <= SA_BLOCKS), "dkv_shared_attention: grid too large");
        const dim3 grid((unsigned)blocks);
        int e;
#define DKV_SA(FF, QQ) e = fast ? sa_launch<FF, QQ, true>(a, grid, st) : sa_launch<FF, QQ, false>(a, grid, st)
        if (f32 && qb) DKV_SA(true, true);
        else if (f32) DKV_SA(true, false);
        else if (qb) DKV_SA(false, true);
        else DKV_SA(false, false);
#undef DKV_SA
        if (e) return e;
        if (a.n_slots == 1) continue;
        if (qb) hipLaunchKernelGGL(shared_merge_kernel<true>, dim3((unsigned)rows), dim3(64 * SM_CLASSES), 0, st, a);
        else hipLaunchKernelGGL(shared_merge_kernel<false>, dim3((unsigned)rows), dim3(64 * SM_CLASSES), 0, st, a);
        if ((e = check_launch("dkv_shared_attention(merge)"))) return e;
    }
    return DKV_OK;
}
