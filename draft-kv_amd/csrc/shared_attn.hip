// Causal attention over a paged full cache whose sequences share pages: the
// keys that the sequences of a group have in common are read once for all of
// them. Reference: the read + softmax of draftkv/llama.py:202-218 (there every
// sequence owns its rows).
//
//     s_k = q . K_k / sqrt(D),  out = sum_k 2^(s_k - m) V_k / sum_k 2^(s_k - m)
//     over the keys k <= position of the row (scores in base 2, m their maximum)
//
// Keys are cut at absolute positions into units of `unit` keys. A row's state
// (m, l, o) over a unit is computed on its own by an online softmax in steps of
// 32 keys, and the merge adds a row's units in an order of their own. So a
// row's result is a function of its keys alone: not of T, of the other rows of
// the call, nor of what is shared. The units that lie whole in a group's
// shared keys are computed for 32 rows of any of its sequences at a time, the
// others for 32 rows of one sequence.
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
#include <algorithm>
#include <type_traits>

#include "dkv_common.h"

// (every instantiation rounds alike, whatever the compiler would fuse in it)
#pragma clang fp contract(off)

namespace dkv {

typedef __bf16 sa_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 sa_bf16x2 __attribute__((ext_vector_type(2)));
typedef float sa_f32x2 __attribute__((ext_vector_type(2)));
typedef float sa_f32x4 __attribute__((ext_vector_type(4)));
typedef float sa_f32x16 __attribute__((ext_vector_type(16)));

constexpr int SA_ROWS = 32, SA_STEP = 32, SA_WAVES = 4;

struct SharedArgs {
    dkv_paged_t c;
    int layer, T, Hq, G;
    int t0, Tn;              // the rows of this launch: t0 .. t0 + Tn - 1 of every sequence
    int unit, n_units;       // keys per unit; units that max_len reaches into
    int n_groups;
    int units_p, tiles_p;    // prefix tasks: units and row tiles per (group, KV head)
    int unit_s, units_s, tiles_s;   // the sequences' own: first unit, units and row tiles per (sequence, KV head)
    int64_t n_prefix, n_tasks;
    const int32_t* first;    // [n_groups + 1]
    const int32_t* shared;   // [batch]
    const void* q;
    const int32_t* start;
    const int32_t* count;
    float qscale;            // log2(e) / sqrt(head_dim)
    float* part;             // o [row of the launch][n_units][D]
    float2* ml;              // (m, l) [row of the launch][n_units]
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

// rows a sequence has after this call, within its block table
__device__ __forceinline__ int sa_len(const SharedArgs& A, int s) {
    return min(A.start[s] + (A.count ? A.count[s] : A.T), A.c.max_blocks * A.c.block_size);
}

// F32: float32 cache. NS: bf16 parts of a query. DP: head_dim rounded up to 32.
// FAST: whole 16-token runs and aligned 16-byte loads.
template <bool F32, bool QBF16, int DP, bool FAST>
__global__ void __launch_bounds__(64 * SA_WAVES, 2) shared_attn_kernel(SharedArgs A) {
    constexpr int NS = QBF16 ? 1 : 3, PS = QBF16 ? 2 : 3;   // bf16 parts of queries and probabilities
    constexpr int DT = DP / 32;
    const dkv_paged_t& c = A.c;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), lane = threadIdx.x % WAVE;
    const int col = lane % 32, half = lane / 32;
    const int D = c.head_dim, bs = c.block_size, G = A.G, H = c.n_kv_heads;

    // ---- the wave's task: a tile of 32 rows of one KV head, and a unit of keys
    int64_t task = (int64_t)blockIdx.x * SA_WAVES + wave;
    if (task >= A.n_tasks) return;
    const bool prefix = task < A.n_prefix;
    int tile, u, h, s0, members;
    if (prefix) {
        tile = (int)(task % A.tiles_p), task /= A.tiles_p;
        u = (int)(task % A.units_p), task /= A.units_p;
        h = (int)(task % H);
        const int g = (int)(task / H);
        s0 = min(max(A.first[g], 0), c.batch), members = min(max(A.first[g + 1], s0), c.batch) - s0;
    } else {
        task -= A.n_prefix;
        tile = (int)(task % A.tiles_s), task /= A.tiles_s;
        u = A.unit_s + (int)(task % A.units_s), task /= A.units_s;
        h = (int)(task % H), s0 = (int)(task / H), members = 1;
    }
    if (members <= 0) return;
    const int per = A.Tn * G;                       // rows of one sequence
    const int n_rows = members * per, r0 = tile * SA_ROWS;
    if (r0 >= n_rows) return;
    // units of the group's shared keys: the prefix tasks', the others' the sequences' own
    const int shared_units = A.units_p ? min(max(min(A.shared[s0], c.max_blocks * bs), 0) / A.unit, A.units_p) : 0;
    if (prefix != (u < shared_units)) return;
    const int k_begin = u * A.unit;

    // ---- the lane's row
    const int r = min(r0 + col, n_rows - 1);
    const bool rvalid = r0 + col < n_rows;
    const int s = s0 + r / per, t = A.t0 + r % per / G, hq = h * G + r % G;
    const int len = sa_len(A, s), last = min(A.start[s] + t, len - 1);   // the row's last key
    const bool live = rvalid && last >= 0;
    const int64_t orow = ((int64_t)s * A.T + t) * A.Hq + hq;
    const int64_t prow = (((int64_t)s * A.Tn + (t - A.t0)) * A.Hq + hq) * A.n_units;
    // the last key that any row of the wave sees, and that all of them see (dead rows see what they like)
    int w_last = live ? last : -1, w_all = live ? last : INT_MAX;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        w_last = max(w_last, __shfl_xor(w_last, o));
        w_all = min(w_all, __shfl_xor(w_all, o));
    }
    w_last = __builtin_amdgcn_readfirstlane(w_last), w_all = __builtin_amdgcn_readfirstlane(w_all);
    const int row_last = live ? last : INT_MAX;
    auto put = [&](int64_t i, float x) {
        if constexpr (QBF16) static_cast<uint16_t*>(A.out)[i] = f32_to_bf16_rne(x);
        else static_cast<float*>(A.out)[i] = x;
    };
    if (u == 0 && rvalid && !live)   // an empty sequence
        for (int d = half; d < D; d += 2) put(orow * D + d, 0.0f);
    if (w_last < k_begin) return;
    // the keys that are there (a prefix unit lies whole in the shared keys)
    const int k_there = prefix ? k_begin + A.unit : min(sa_len(A, s0), k_begin + A.unit);
    const int k_end = min(k_there, w_last + 1);

    // ---- queries: B operands
    constexpr int KS = F32 ? DP / 8 : DP / 16;
    sa_bf16x8 qp[F32 ? 1 : KS][NS];
    sa_f32x4 qf[F32 ? KS : 1];
    {
        auto at = [&](int d) -> float { return d < D ? load_elem(A.q, orow * D + d, QBF16 ? DKV_BF16 : DKV_F32) : 0.0f; };
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) qf[j][e] = at(8 * j + 4 * half + e) * A.qscale;
        } else {
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float x = at(16 * j + 8 * half + e), y = at(16 * j + 8 * half + e + 1);
                    // (bf16 queries stay whole: their scores are scaled)
                    if constexpr (NS == 1) sa_split<NS>(x, y, qp[j], e);
                    else sa_split<NS>(x * A.qscale, y * A.qscale, qp[j], e);
                }
        }
    }

    const int32_t* btab = c.block_table + ((int64_t)s0 * c.n_layers + A.layer) * c.max_blocks;
    const int64_t bel = paged_block_elems(c);
    const int key_of = (col & 0x13) | (col & 4) << 1 | (col & 8) >> 1;   // bits 2 and 3 exchanged

    sa_f32x16 acc[DT];
    float m_run, l_run;
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][e] = 0.0f;
        m_run = -INFINITY, l_run = 0.0f;
    };

    // One walk over the unit, K and V straight from memory. Careful: values that are not finite, one by one.
    auto walk = [&](auto careful) {
      constexpr bool CAREFUL = decltype(careful)::value;
      clear();
      for (int kb = k_begin; kb < k_end; kb += SA_STEP) {
        // ---- K and V operands of 32 keys
        float kf[F32 ? KS : 1][4];
        sa_bf16x8 kr[F32 ? 1 : KS];
        float vf[F32 ? DT : 1][2][8];
        sa_bf16x8 vr[F32 ? 1 : DT][2];
        const int last_there = k_there - 1;
        if constexpr (FAST) {
            const int p0 = kb, p1 = min(kb + 16, last_there & ~15);   // two runs of 16 tokens
            const int32_t b0 = __builtin_amdgcn_readfirstlane(btab[p0 / bs]), b1 = __builtin_amdgcn_readfirstlane(btab[p1 / bs]);
            const int64_t g0 = b0 * bel, g1 = b1 * bel;
            const int64_t kat = (key_of < 16 ? g0 : g1) + ((int64_t)h * bs + (key_of < 16 ? p0 : p1) % bs + key_of % 16) * DP;
            const int64_t vrow = (int64_t)H * bs * DP + ((int64_t)h * DP + col) * bs + 8 * half;
            if constexpr (F32) {
                const float* pool = static_cast<const float*>(c.pool);
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    const sa_f32x4 x = *reinterpret_cast<const sa_f32x4*>(pool + kat + 8 * j + 4 * half);
#pragma unroll
                    for (int e = 0; e < 4; ++e) kf[j][e] = x[e];
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const sa_f32x4 w = *reinterpret_cast<const sa_f32x4*>(
                                pool + (x ? g1 : g0) + vrow + (int64_t)32 * dt * bs + (x ? p1 : p0) % bs + 4 * y);
#pragma unroll
                            for (int e = 0; e < 4; ++e) vf[dt][x][4 * y + e] = w[e];
                        }
            } else {
                const uint16_t* pool = static_cast<const uint16_t*>(c.pool);
#pragma unroll
                for (int j = 0; j < KS; ++j) kr[j] = *reinterpret_cast<const sa_bf16x8*>(pool + kat + 16 * j + 8 * half);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        vr[dt][x] = *reinterpret_cast<const sa_bf16x8*>(pool + (x ? g1 : g0) + vrow + (int64_t)32 * dt * bs +
                                                                        (x ? p1 : p0) % bs);
            }
        } else {
            const int kp = min(kb + key_of, last_there);
            const int32_t kblk = btab[kp / bs];
            auto kelem = [&](int d) { return d < D ? load_elem(c.pool, paged_k_off(c, kblk, kp % bs, h, d), c.dtype) : 0.0f; };
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < KS; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) kf[j][e] = kelem(8 * j + 4 * half + e);
            } else {
#pragma unroll
                for (int j = 0; j < KS; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) kr[j][e] = (__bf16)kelem(16 * j + 8 * half + e);
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int vp = min(kb + 16 * x + 8 * half + e, last_there);
                    const int32_t vblk = btab[vp / bs];
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const int d = 32 * dt + col;
                        const float w = d < D ? load_elem(c.pool, paged_v_off(c, vblk, vp % bs, h, d), c.dtype) : 0.0f;
                        if constexpr (F32) vf[dt][x][e] = w;
                        else vr[dt][x][e] = (__bf16)w;
                    }
                }
        }
        // ---- scores: lane holds keys kb + 16 x + 8 half + e of its row at 8 x + e
        sa_f32x16 sc;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = 0.0f;
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j][e], qf[j][e], sc, 0, 0, 0);
        } else {
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
                for (int i = 0; i < NS; ++i) sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kr[j], qp[j][i], sc, 0, 0, 0);
        }
        float p[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) p[k] = !F32 && NS == 1 ? sc[k] * A.qscale : sc[k];
        const bool masked = kb + SA_STEP - 1 > w_all || kb + SA_STEP > k_there;   // uniform
        const int k_lane = kb + 8 * half;
        if constexpr (CAREFUL && !F32 && NS > 1) {
            // An infinity times a query's parts is no number where they differ in sign or one is 0: its score again,
            // channel by channel.
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                if (p[k] == p[k]) continue;
                const int kp = min(k_lane + 16 * (k / 8) + k % 8, k_there - 1);
                const int32_t blk = btab[kp / bs];
                float x = 0.0f;
                for (int d = 0; d < D; ++d)
                    x += load_elem(A.q, orow * D + d, DKV_F32) * A.qscale * load_elem(c.pool, paged_k_off(c, blk, kp % bs, h, d), c.dtype);
                p[k] = x;
            }
        }
        if (masked) {
            const int lim = min(row_last, k_there - 1);
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (k_lane + 16 * (k / 8) + k % 8 > lim) p[k] = -INFINITY;
        }
        float mx = p[0];
#pragma unroll
        for (int k = 1; k < 16; ++k) mx = fmaxf(mx, p[k]);
        const float m_new = fmaxf(m_run, sa_max_halves(mx));
        const float ms = m_new == -INFINITY ? 0.0f : m_new;   // a row that sees no key yet: p = 0
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            p[k] = sa_exp2(p[k] - ms);
            sum += p[k];
        }
        const float alpha = m_new == m_run ? 1.0f : sa_exp2(m_run - m_new);
        l_run = l_run * alpha + sum;
        m_run = m_new;
        if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][e] *= alpha;
        }
        // ---- V past the cache's end: zero (whatever the page holds, 0 * it could be NaN)
        if (kb + SA_STEP > k_there) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (k_lane + 16 * x + e >= k_there)
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            if constexpr (F32) vf[dt][x][e] = 0.0f;
                            else vr[dt][x][e] = (__bf16)0.0f;
                        }
        }
        if constexpr (CAREFUL) {   // infinities and NaN of V: out of the product, to the rows that see them by hand
            for (int x = 0; x < 2; ++x)
                for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float pk = 0.0f;
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const float z = __shfl(p[8 * y + e], col + 32 * hh);
                            pk = y == x ? z : pk;
                        }
                        const bool sees = kb + 16 * x + 8 * hh + e <= row_last;
#pragma unroll
                        for (int dt = 0; dt < DT; ++dt) {
                            float w = 0.0f;
#pragma unroll
                            for (int y = 0; y < 2; ++y)
                                if (y == x) {
                                    if constexpr (F32) w = vf[dt][y][e];
                                    else w = (float)vr[dt][y][e];
                                }
                            if (!__any(!(fabsf(w) < INFINITY))) continue;
#pragma unroll
                            for (int k = 0; k < 16; ++k) {   // the lane's channels of this tile
                                const float v = __shfl(w, 8 * (k / 4) + 4 * half + k % 4 + 32 * hh);
                                if (sees && !(fabsf(v) < INFINITY)) acc[dt][k] += pk * v;
                            }
                        }
                    }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if constexpr (F32) {
                            if (!(fabsf(vf[dt][x][e]) < INFINITY)) vf[dt][x][e] = 0.0f;
                        } else {
                            if (!(fabsf((float)vr[dt][x][e]) < INFINITY)) vr[dt][x][e] = (__bf16)0.0f;
                        }
                    }
        }
        // ---- O^T += V^T . P^T
        if constexpr (F32) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
                        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(vf[dt][x][e], p[8 * x + e], acc[dt], 0, 0, 0);
        } else {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                sa_bf16x8 pp[PS];
#pragma unroll
                for (int e = 0; e < 8; e += 2) sa_split<PS>(p[8 * x + e], p[8 * x + e + 1], pp, e);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                    for (int i = 0; i < PS; ++i)
                        acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vr[dt][x], pp[i], acc[dt], 0, 0, 0);
            }
        }
      }
    };
    walk(std::false_type{});
    // A NaN: of a key that its row sees, or 0 times what it does not. Again, and telling them apart.
    bool odd = l_run != l_run;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int k = 0; k < 16; ++k) odd |= acc[dt][k] != acc[dt][k];
    if (__any(odd)) walk(std::true_type{});
    // ---- out: channels 32 dt + 8 (k / 4) + 4 half + k % 4 of the lane's row
    const float l = sa_sum_halves(l_run);
    if (!live) return;
    const bool alone = last < A.unit || A.n_units == 1;   // the row sees one unit
    if (alone && u > 0) return;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int d = 32 * dt + 8 * (k / 4) + 4 * half + k % 4;
            if (d >= D) continue;
            if (alone) put(orow * D + d, acc[dt][k] / l);
            else A.part[(prow + u) * D + d] = acc[dt][k];
        }
    if (!alone && half == 0) A.ml[prow + u] = make_float2(m_run, l);
}

// Merge of each row's units: their common maximum first, then the weighted
// sums, units u, u + 4, ... in order and these four last, so the result depends
// on the row's units alone. A wave per row and class.
constexpr int SM_CLASSES = 4;
template <bool QBF16>
__global__ void __launch_bounds__(64 * SM_CLASSES) shared_merge_kernel(SharedArgs A) {
    const int w = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, D = A.c.head_dim;
    int64_t i = blockIdx.x;
    const int hq = (int)(i % A.Hq);
    i /= A.Hq;
    const int t = A.t0 + (int)(i % A.Tn), s = (int)(i / A.Tn);
    const int last = min(A.start[s] + t, sa_len(A, s) - 1);
    const int n = last < 0 ? 0 : min(last / A.unit + 1, A.n_units);
    if (n <= 1) return;   // the attention kernel wrote the row
    const int64_t prow = (int64_t)blockIdx.x * A.n_units;
    float m = -INFINITY;
    for (int u = lane; u < n; u += WAVE) m = fmaxf(m, A.ml[prow + u].x);
    m = wave_max(m);
    const float ms = m == -INFINITY ? 0.0f : m;
    const int c0 = min(lane, D - 1), c1 = min(lane + WAVE, D - 1);
    float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int u = w; u < n; u += SM_CLASSES) {
        const float2 x = A.ml[prow + u];
        const float f = sa_exp2(x.x - ms);
        l = fmaf(x.y, f, l);
        o0 = fmaf(A.part[(prow + u) * D + c0], f, o0);
        o1 = fmaf(A.part[(prow + u) * D + c1], f, o1);
    }
    __shared__ float sl[SM_CLASSES], so[SM_CLASSES][2][WAVE];
    if (lane == 0) sl[w] = l;
    so[w][0][lane] = o0, so[w][1][lane] = o1;
    __syncthreads();
    if (w > 1 || lane + WAVE * w >= D) return;
    float lt = 0.0f, ot = 0.0f;
#pragma unroll
    for (int k = 0; k < SM_CLASSES; ++k) lt += sl[k], ot += so[k][w][lane];
    const int64_t at = (((int64_t)s * A.T + t) * A.Hq + hq) * D + lane + WAVE * w;
    if constexpr (QBF16) static_cast<uint16_t*>(A.out)[at] = f32_to_bf16_rne(ot / lt);
    else static_cast<float*>(A.out)[at] = ot / lt;
}

// Rows per launch: as many of the T as keep the partials within this
constexpr size_t SA_WORK_BYTES = (size_t)512 << 20;
static size_t sa_row_bytes(const dkv_paged_t& c, int Hq, int n_units) {   // of one t
    return sizeof(float) * (size_t)c.batch * Hq * n_units * (c.head_dim + 2);
}
static int sa_rows(const dkv_paged_t& c, int T, int Hq, int n_units) {
    return (int)std::min<size_t>(T, std::max<size_t>(1, SA_WORK_BYTES / sa_row_bytes(c, Hq, n_units)));
}
static int sa_units(const dkv_paged_t& c, int max_len, int unit) {
    const int64_t keys = std::min<int64_t>(max_len, (int64_t)c.max_blocks * c.block_size);
    return (int)((keys + unit - 1) / unit);
}

template <bool F32, bool QBF16, bool FAST>
static void sa_launch(const SharedArgs& a, dim3 grid, hipStream_t st) {
    const dim3 blk(64 * SA_WAVES);
    switch ((a.c.head_dim + 31) / 32) {
        case 1: hipLaunchKernelGGL((shared_attn_kernel<F32, QBF16, 32, FAST>), grid, blk, 0, st, a); break;
        case 2: hipLaunchKernelGGL((shared_attn_kernel<F32, QBF16, 64, FAST>), grid, blk, 0, st, a); break;
        case 3: hipLaunchKernelGGL((shared_attn_kernel<F32, QBF16, 96, FAST>), grid, blk, 0, st, a); break;
        default: hipLaunchKernelGGL((shared_attn_kernel<F32, QBF16, 128, FAST>), grid, blk, 0, st, a); break;
    }
}

static int sa_check(const dkv_paged_t& c, const dkv_groups_t& g, int T, int Hq, int max_len, int unit) {
    DKV_REQUIRE(c.dtype == DKV_F32 || c.dtype == DKV_BF16, "dkv_shared_attention: bad cache dtype");
    DKV_REQUIRE(c.batch > 0 && c.n_layers > 0 && c.n_kv_heads > 0 && c.block_size > 0 && c.max_blocks > 0,
                "dkv_shared_attention: bad cache shape");
    DKV_REQUIRE((int64_t)c.max_blocks * c.block_size < (1LL << 31) - (1 << 16), "dkv_shared_attention: more than 2^31 positions");
    DKV_REQUIRE(c.head_dim > 0 && c.head_dim <= 128, "dkv_shared_attention: head_dim must be 1..128");
    DKV_REQUIRE(Hq > 0 && Hq % c.n_kv_heads == 0, "dkv_shared_attention: query heads must be a multiple of KV heads");
    DKV_REQUIRE(unit > 0 && unit % SA_STEP == 0, "dkv_shared_attention: unit_keys must be a multiple of 32");
    DKV_REQUIRE(max_len > 0, "dkv_shared_attention: max_len must be > 0");
    DKV_REQUIRE(T >= 0 && (int64_t)c.batch * T * Hq < (1LL << 31), "dkv_shared_attention: too many rows");
    DKV_REQUIRE(g.n_groups >= 0 && g.n_groups <= c.batch, "dkv_shared_attention: n_groups must lie in 0..batch");
    DKV_REQUIRE(g.n_groups == 0 || (g.max_members > 0 && g.max_members <= c.batch && g.min_shared >= 0 &&
                                    g.min_shared <= g.max_shared),
                "dkv_shared_attention: bad group bounds");
    return DKV_OK;
}

}  // namespace dkv

extern "C" size_t dkv_shared_attention_workspace(const dkv_paged_t* cache, int32_t T, int32_t n_q_heads, int32_t max_len,
                                                 int32_t unit_keys) {
    if (!cache || T <= 0 || n_q_heads <= 0 || max_len <= 0 || unit_keys <= 0 || cache->batch <= 0) return 0;
    const int n = dkv::sa_units(*cache, max_len, unit_keys);
    if (n <= 1) return 0;
    return dkv::sa_rows(*cache, T, n_q_heads, n) * dkv::sa_row_bytes(*cache, n_q_heads, n) + 8;   // (m, l) on 8 bytes
}

extern "C" int dkv_shared_attention(const dkv_paged_t* cache, const dkv_groups_t* groups, int32_t layer, const void* q,
                                    int32_t q_dtype, int32_t T, int32_t n_q_heads, const int32_t* start,
                                    const int32_t* count, int32_t max_len, int32_t unit_keys, void* out, void* work,
                                    size_t work_bytes, dkv_stream_t stream) {
    using namespace dkv;
    DKV_REQUIRE(cache && groups, "dkv_shared_attention: NULL argument");
    const dkv_paged_t c = *cache;
    const dkv_groups_t g = *groups;
    const int rc = sa_check(c, g, T, n_q_heads, max_len, unit_keys);
    if (rc) return rc;
    DKV_REQUIRE(layer >= 0 && layer < c.n_layers, "dkv_shared_attention: layer out of range");
    DKV_REQUIRE(q_dtype == DKV_F32 || q_dtype == DKV_BF16, "dkv_shared_attention: bad query dtype");
    if (T == 0) return DKV_OK;
    DKV_REQUIRE(q && start && out && c.pool && c.block_table && (g.n_groups == 0 || (g.first && g.shared)),
                "dkv_shared_attention: NULL argument");
    SharedArgs a = {};
    a.c = c, a.layer = layer, a.T = T, a.Hq = n_q_heads, a.G = n_q_heads / c.n_kv_heads;
    a.unit = unit_keys, a.n_units = sa_units(c, max_len, unit_keys);
    a.n_groups = g.n_groups, a.first = g.first, a.shared = g.shared;
    a.q = q, a.start = start, a.count = count, a.out = out;
    a.qscale = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(c.head_dim)));
    const size_t need = dkv_shared_attention_workspace(cache, T, n_q_heads, max_len, unit_keys);
    if (need && (!work || work_bytes < need))
        return fail(DKV_EWORKSPACE, "dkv_shared_attention: workspace too small (need " + std::to_string(need) + ")");
    const int step = sa_rows(c, T, n_q_heads, a.n_units);
    hipStream_t st = as_stream(stream);
    const bool f32 = c.dtype == DKV_F32, qb = q_dtype == DKV_BF16;
    const bool fast = c.block_size % 16 == 0 && c.head_dim % 32 == 0 && reinterpret_cast<uintptr_t>(c.pool) % 16 == 0;
    for (a.t0 = 0; a.t0 < T; a.t0 += step) {
        a.Tn = std::min(step, T - a.t0);
        const int64_t rows = (int64_t)c.batch * a.Tn * n_q_heads;
        a.part = static_cast<float*>(work);
        a.ml = reinterpret_cast<float2*>(a.part + (rows * a.n_units * c.head_dim + 1) / 2 * 2);
        const int64_t per = (int64_t)a.Tn * a.G;
        a.units_p = g.n_groups ? std::min(g.max_shared / unit_keys, a.n_units) : 0;
        a.tiles_p = (int)((g.max_members * per + SA_ROWS - 1) / SA_ROWS);
        a.unit_s = g.n_groups ? std::min(g.min_shared / unit_keys, a.n_units - 1) : 0;
        a.units_s = a.n_units - a.unit_s;
        a.tiles_s = (int)((per + SA_ROWS - 1) / SA_ROWS);
        a.n_prefix = (int64_t)a.n_groups * c.n_kv_heads * a.units_p * a.tiles_p;
        a.n_tasks = a.n_prefix + (int64_t)c.batch * c.n_kv_heads * a.units_s * a.tiles_s;
        const int64_t blocks = (a.n_tasks + SA_WAVES - 1) / SA_WAVES;
        DKV_REQUIRE(blocks < (1LL << 31), "dkv_shared_attention: grid too large");
        const dim3 grid((unsigned)blocks);
#define DKV_SA(FF, QQ)                                    \
    do {                                                  \
        if (fast) sa_launch<FF, QQ, true>(a, grid, st);   \
        else sa_launch<FF, QQ, false>(a, grid, st);       \
    } while (0)
        if (f32 && qb) DKV_SA(true, true);
        else if (f32) DKV_SA(true, false);
        else if (qb) DKV_SA(false, true);
        else DKV_SA(false, false);
#undef DKV_SA
        if (const int e = check_launch("dkv_shared_attention")) return e;
        if (a.n_units == 1) continue;
        if (qb) hipLaunchKernelGGL(shared_merge_kernel<true>, dim3((unsigned)rows), dim3(64 * SM_CLASSES), 0, st, a);
        else hipLaunchKernelGGL(shared_merge_kernel<false>, dim3((unsigned)rows), dim3(64 * SM_CLASSES), 0, st, a);
        if (const int e = check_launch("dkv_shared_attention(merge)")) return e;
    }
    return DKV_OK;
}
