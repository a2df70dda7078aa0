// Beam search's selection: of the continuations of a prompt's beams the k best
// (no counterpart in the reference, which decodes one sequence,
// draftkv/engine.py:108-119).
//
//     score(b, v) = cum_b + (x_bv - lse_b),  lse_b = m_b + log sum_v exp(x_bv - m_b)      (float64)
//
// in the order (score, lowest beam, largest logit, lowest token). A row that
// holds NaN or +infinity, or nothing but -infinity, has no continuations, nor
// has a beam whose cum is -infinity or NaN.
//
// Two launches:
//   1. scan    grid (segment, row): the row's tiles of 8192 logits, in
//              registers: each wave's maximum and float64 sum of exponentials,
//              and a list of logits with the segment's k largest.
//   2. select  one workgroup per prompt: each row's lse and k largest, a wave
//              per row, then the k best of all rows (a rank is a binary
//              search in every other row).
// Bound: 256 rows of 128256 take 51 us in all, 38 of them the scan: 131 MB of
// float32 logits at 3.4 TB/s, and 50 us with bf16 logits, so it is the
// float64 exponentials and the ranking (30 VALU instructions per logit, the
// VALU busy two thirds of the time), not the bytes. 32 rows 18 us, four of 49152 16: two dependent launches of 7
// and 7 (the select: one workgroup per prompt, a chain of loads, two ranks).
// One instance for every k: a scan whose lists were sized for k up to 32 (twice
// the workgroups per CU) took 52, 18.5 and 15.7.
#include <algorithm>

#include "dexp.h"

namespace dkv {

constexpr int BEAM_THREADS = 256, BEAM_PER = 32;
constexpr int BEAM_TILE = BEAM_THREADS * BEAM_PER;
constexpr int BEAM_MAX_K = 64, BEAM_MAX_LIST = 4096, BEAM_MAX_ROW_LIST = 1024;
constexpr int BEAM_SEL_THREADS = 512;

struct BeamTile {   // of the logits of one wave in a tile
    double sum;   // of exp(x - mx)
    float mx;
    int bad;      // NaN or +infinity among them
};
constexpr int BEAM_PARTS = BEAM_THREADS / WAVE;   // per tile

struct BeamArgs {
    const void* x;
    const double* cum;
    int64_t stride;              // elements between rows
    int vocab, beams, k, n_tiles, segs, per_seg;   // tiles per segment
    int list;                    // keys that a segment's list holds
    BeamTile* tiles;             // [row][n_tiles][BEAM_PARTS]
    uint64_t* lists;             // [row][segs][list] keys, in any order: its k best among them
    uint2* heads;                // [row][segs] how many, and a logit (ordered) that k of them reach
    double* out_score;
    int32_t* out_parent;
    int32_t* out_token;
};

// A logit and its index as one number: larger logits first, lower indices first among equal ones.
__device__ __forceinline__ uint64_t beam_key(float x, int i) {
    const uint32_t u = __float_as_uint(x + 0.0f);   // (-0 becomes the 0 that it is equal to)
    const uint32_t o = (u >> 31) ? ~u : u | 0x80000000u;
    return (uint64_t)o << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float beam_logit(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int beam_token(uint64_t key) { return (int)~(uint32_t)key; }

// The thread's logits of a tile: element 4 (t + 256 j) + e in register 4 j + e, -infinity past the row.
template <bool BF16, bool VEC, bool WHOLE>
__device__ __forceinline__ void beam_load_tile(const void* base, int i0, int n, float (&v)[BEAM_PER]) {
#pragma unroll
    for (int j = 0; j < BEAM_PER / 4; ++j) {
        const int i = i0 + 4 * ((int)threadIdx.x + BEAM_THREADS * j);
        if constexpr (VEC) {   // n % 4 == 0: four logits are whole or past the end
            if constexpr (BF16) {
                const uint2 w = WHOLE || i < n ? *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i)
                                      : make_uint2(0xff80ff80u, 0xff80ff80u);
                v[4 * j] = __uint_as_float(w.x << 16), v[4 * j + 1] = __uint_as_float(w.x & 0xffff0000u);
                v[4 * j + 2] = __uint_as_float(w.y << 16), v[4 * j + 3] = __uint_as_float(w.y & 0xffff0000u);
            } else {
                const float4 w = WHOLE || i < n ? *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i)
                                       : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                v[4 * j] = w.x, v[4 * j + 1] = w.y, v[4 * j + 2] = w.z, v[4 * j + 3] = w.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * j + e] = WHOLE || i + e < n ? load_elem(base, i + e, BF16 ? DKV_BF16 : DKV_F32) : -INFINITY;
        }
    }
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void beam_load(const void* base, int i0, int n, float (&v)[BEAM_PER]) {
    if (i0 + BEAM_TILE <= n) beam_load_tile<BF16, VEC, true>(base, i0, n, v);
    else beam_load_tile<BF16, VEC, false>(base, i0, n, v);
}

// Over the wave by lane moves of the VALU (an LDS permute per step takes ten times as long); the result is uniform.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t beam_dpp(uint32_t old, uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, ROWS, 0xf, false);
}
template <class F>
__device__ __forceinline__ uint32_t beam_reduce(uint32_t v, F f) {   // f(x, x) = x
    v = f(v, beam_dpp<0x111, 0xf>(v, v));   // from the lane before, 2, 4, 8 before in rows of 16,
    v = f(v, beam_dpp<0x112, 0xf>(v, v));
    v = f(v, beam_dpp<0x114, 0xf>(v, v));
    v = f(v, beam_dpp<0x118, 0xf>(v, v));
    v = f(v, beam_dpp<0x142, 0xa>(v, v));   // the rows' last lanes to the next rows
    v = f(v, beam_dpp<0x143, 0xc>(v, v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, WAVE - 1);
}
__device__ __forceinline__ uint32_t beam_wave_max(uint32_t v) {
    return beam_reduce(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ float beam_wave_max(float v) {
    return __uint_as_float(beam_reduce(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double beam_add_dpp(double v) {
    return v + __hiloint2double((int)beam_dpp<CTRL, ROWS>(0, (uint32_t)__double2hiint(v)), (int)beam_dpp<CTRL, ROWS>(0, (uint32_t)__double2loint(v)));
}
__device__ __forceinline__ double beam_wave_sum(double v) {
    v = beam_add_dpp<0x111, 0xf>(v);
    v = beam_add_dpp<0x112, 0xf>(v);
    v = beam_add_dpp<0x114, 0xf>(v);
    v = beam_add_dpp<0x118, 0xf>(v);
    v = beam_add_dpp<0x142, 0xa>(v);
    v = beam_add_dpp<0x143, 0xc>(v);
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), WAVE - 1), __builtin_amdgcn_readlane(__double2loint(v), WAVE - 1));
}

// floats in order as unsigned numbers
__device__ __forceinline__ uint32_t beam_order(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float beam_max3(float a, float b, float c) {   // (fmaxf would quiet each operand first)
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// The r-th largest of the wave's distinct values. Few: of 16 groups of four lanes (a bound from below that is as good for a
// small r, at a quarter of the instructions).
__device__ __forceinline__ uint32_t beam_nth(uint32_t v, int r) {
    int rank = 0;
    if (r <= 4) {
        v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));   // lanes exchanged in pairs,
        v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));   // and pairs in quads
#pragma unroll
        for (int i = 0; i < WAVE; i += 4) rank += (uint32_t)__builtin_amdgcn_readlane((int)v, i) > v;
    } else {
#pragma unroll 16
        for (int i = 0; i < WAVE; ++i) rank += (uint32_t)__builtin_amdgcn_readlane((int)v, i) > v;
    }
    return (uint32_t)__builtin_amdgcn_readlane((int)v, __ffsll((unsigned long long)__ballot(rank == r - 1)) - 1);
}

// What a logit must reach to be ranked: of the threads' largest, the ceil(k / 4)-th of
// each of the four waves, and of those the least (k logits are as large), or what an earlier tile of the segment asked for.
// Rows of model logits pass little more than k per tile that way. Each wave lists its own; the lists are ranked when one is
// half full, and at the end. A tile that overflows one (equal logits) takes the k-th of all threads' largest by value and
// index, which at most k threads' logits pass.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(BEAM_THREADS, 3) beam_scan_kernel(BeamArgs A) {
    constexpr int KM = BEAM_MAX_K;
    constexpr int NW = BEAM_THREADS / WAVE;
    constexpr int CAP = KM * BEAM_PER / NW + KM;    // a wave's list; all of them hold k threads' logits and the k best before
    __shared__ double tab[EXP_TAB];
    static_assert(CAP % 8 == 0, "lists are read 8 keys at a time");
    __shared__ __align__(16) uint64_t cand[NW * CAP];
    __shared__ uint64_t best[KM], tmax[BEAM_THREADS];
    __shared__ uint32_t wthr[NW];
    __shared__ int n_cand[NW], n_flat;
    __shared__ uint64_t s_thr;
    const int seg = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid % WAVE, w = tid / WAVE;
    const int k = A.k, kq = (k + NW - 1) / NW;
    const char* base = static_cast<const char*>(A.x) + (int64_t)row * A.stride * (BF16 ? 2 : 4);
    const int t0 = seg * A.per_seg, t1 = min(t0 + A.per_seg, A.n_tiles);
    load_exp_tab(tab);
    // The k best of the waves' lists (list i: n[i] from i * CAP on) in order to best[]; how many there are. Ends behind a
    // barrier.
    auto rank_lists = [&](const int (&n)[NW]) {
#pragma unroll
        for (int a = 0; a < NW; ++a)   // to whole 8s: keys in flight together
            if (tid < (-n[a] & 7)) cand[a * CAP + n[a] + tid] = 0;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int a = 0; a < NW; ++a) {
            total += n[a];
            for (int i = tid; i < n[a]; i += BEAM_THREADS) {
                const uint64_t key = cand[a * CAP + i];
                int rank = 0;
#pragma unroll
                for (int b = 0; b < NW; ++b)
                    for (int j = 0; j < n[b]; j += 8)
#pragma unroll
                        for (int e = 0; e < 8; ++e) rank += cand[b * CAP + j + e] > key;
                if (rank < k) best[rank] = key;
            }
        }
        __syncthreads();
        return min(total, k);
    };
    uint32_t floor = 0;   // (uniform) what the tiles so far ask for
    int mine_n = 0;       // (of the wave) its list's length
    int have[NW] = {};    // (uniform) the lists' lengths before the tile
    for (int tile = t0; tile < t1; ++tile) {
        const int i0 = tile * BEAM_TILE;
        float v[BEAM_PER];
        beam_load<BF16, VEC>(base, i0, A.vocab, v);
        float mx = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < BEAM_PER; j += 2) {
            bad |= __builtin_isunordered(v[j], v[j + 1]);
            mx = beam_max3(mx, v[j], v[j + 1]);
        }
        const float wm = beam_wave_max(mx);
        bad |= wm == INFINITY;
        // the kq-th of the wave's threads' largest, but for its last 6 bits; nothing where few pass what was asked for
        const uint32_t mine = (beam_order(mx) & ~63u) | (63 - lane);
        uint32_t nth = 0;
        if (__popcll(__ballot(mine > floor)) >= 2 * kq) nth = beam_nth(mine, kq) & ~63u;
        if (lane == 0) wthr[w] = nth;
        __syncthreads();
        uint32_t thr = wthr[0];
#pragma unroll
        for (int i = 1; i < NW; ++i) thr = min(thr, wthr[i]);
        floor = max(floor, thr);
        const float thr_x = floor <= 0x007fffffu ? -INFINITY : __uint_as_float((floor >> 31) ? floor & 0x7fffffffu : ~floor);   // (that is -infinity, and below)
#pragma unroll
        for (int j = 0; j < BEAM_PER; ++j) {
            const uint64_t in = __ballot(v[j] >= thr_x);
            if (in) {   // few
                const bool mine = v[j] >= thr_x && v[j] > -INFINITY;
                const uint64_t live = __ballot(mine);
                const int at = mine_n + __popcll(live & ((1ull << lane) - 1));
                if (mine && at < CAP) cand[w * CAP + at] = beam_key(v[j], i0 + 4 * (tid + BEAM_THREADS * (j / 4)) + j % 4);
                mine_n += __popcll(live);
            }
        }
        if (lane == 0) n_cand[w] = mine_n;
        // ---- exponentials: of the wave's logits, below their maximum
        const double m = wm == -INFINITY ? 0.0 : (double)wm;
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < BEAM_PER; j += 4) {
            double y[4], ex[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = fmax((double)v[j + e] - m, -708.0);   // (less adds 1e-307 of the sum)
            dexp_sum_n<4>(y, ex, tab);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum += ex[e];
        }
        sum = beam_wave_sum(sum);
        const bool wbad = __any(bad);
        if (lane == 0) A.tiles[((int64_t)row * A.n_tiles + tile) * NW + w] = BeamTile{sum, wm, wbad};
        __syncthreads();
        int now[NW], most = 0;
#pragma unroll
        for (int i = 0; i < NW; ++i) now[i] = n_cand[i], most = max(most, now[i]);
        if (most <= CAP / 2) {   // uniform
#pragma unroll
            for (int i = 0; i < NW; ++i) have[i] = now[i];
            continue;
        }
        // ---- the lists so far to their k best, in the first one
        const bool over = most > CAP;
        const int n_best = rank_lists(over ? have : now);
        if (tid < n_best) cand[tid] = best[tid];
        if (tid == 0) n_flat = n_best, s_thr = 0;
        if (n_best == k) floor = max(floor, (uint32_t)(best[k - 1] >> 32));
        if (over) {   // and this tile's again, by value and index
            float mx = -INFINITY;
            int arg = 0;
#pragma unroll
            for (int j = 0; j < BEAM_PER; ++j)
                if (v[j] > mx) mx = v[j], arg = j;   // (indices rise with j)
            const uint64_t mine = mx > -INFINITY ? beam_key(mx, i0 + 4 * (tid + BEAM_THREADS * (arg / 4)) + arg % 4) : 0;
            tmax[tid] = mine;
            __syncthreads();
            int rank = 0;
            for (int i = 0; i < BEAM_THREADS; ++i) rank += tmax[i] > mine;
            if (rank == k - 1) s_thr = mine;
            __syncthreads();
            const uint64_t exact = s_thr;
            for (int j = 0; j < BEAM_PER; ++j) {
                float x = v[0];
#pragma unroll
                for (int e = 1; e < BEAM_PER; ++e) x = j == e ? v[e] : x;
                const uint64_t key = beam_key(x, i0 + 4 * (tid + BEAM_THREADS * (j / 4)) + j % 4);
                if (key >= exact && x > -INFINITY) cand[atomicAdd(&n_flat, 1)] = key;
            }
            __syncthreads();
            // (as one list from the start: k + 32 k entries at most)
            const int n = n_flat;
            for (int i = tid; i < n; i += BEAM_THREADS) {
                const uint64_t key = cand[i];
                int rank = 0;
                for (int j = 0; j < n; ++j) rank += cand[j] > key;
                if (rank < k) best[rank] = key;
            }
            __syncthreads();
            const int n_best = min(n, k);
            if (tid < n_best) cand[tid] = best[tid];
            if (tid == 0) n_flat = n_best;
            if (n_best == k) floor = max(floor, (uint32_t)(best[k - 1] >> 32));
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NW; ++i) have[i] = i == 0 ? n_flat : 0;
        mine_n = w == 0 ? have[0] : 0;
    }
    // ---- the lists out, without what the last floor leaves out; where that is too much, the k best
    const int64_t at = (int64_t)row * A.segs + seg;
    uint64_t* out = A.lists + at * A.list;
    int n = 0;
    for (int i = lane; i - lane < have[w]; i += WAVE) {   // (whole waves)
        const uint64_t key = i < have[w] ? cand[w * CAP + i] : 0;
        const uint64_t in = __ballot((uint32_t)(key >> 32) >= floor && key != 0);
        if (in >> lane & 1) cand[w * CAP + n + __popcll(in & ((1ull << lane) - 1))] = key;   // (at or before where it was)
        n += __popcll(in);
    }
    if (lane == 0) n_cand[w] = n;   // (a wave still reading the lengths of the last tile uses its own alone)
    __syncthreads();
    int first = 0, total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        have[i] = n_cand[i];
        first += i < w ? have[i] : 0;
        total += have[i];
    }
    if (total <= A.list) {
        for (int i = lane; i < n; i += WAVE) out[first + i] = cand[w * CAP + i];
    } else {
        total = rank_lists(have);
        for (int i = tid; i < total; i += BEAM_THREADS) out[i] = best[i];
    }
    if (tid == 0) A.heads[at] = make_uint2(total, floor);
}

__global__ void __launch_bounds__(BEAM_SEL_THREADS) beam_select_kernel(BeamArgs A) {
    extern __shared__ __align__(16) char lds[];
    const int B = A.beams, k = A.k, n_list = A.segs * A.list;
    constexpr int NW = BEAM_SEL_THREADS / WAVE;
    uint64_t* rows = reinterpret_cast<uint64_t*>(lds);             // [B][k] the rows' largest logits
    double* score = reinterpret_cast<double*>(rows + B * k);       // [B][k] and their scores
    uint64_t* lists = reinterpret_cast<uint64_t*>(score + B * k);  // [NW][segs * list]
    int* n_row = reinterpret_cast<int*>(lists + NW * n_list);   // [B] live continuations of a row
    const int p = blockIdx.x, tid = threadIdx.x, lane = tid % WAVE, w = tid / WAVE;
    for (int b = w; b < B; b += NW) {
        const int64_t row = (int64_t)p * B + b;
        const uint64_t* from = A.lists + row * n_list;
        uint64_t* mine = lists + w * n_list;
        const BeamTile* t = A.tiles + row * A.n_tiles * BEAM_PARTS;
        const int n_parts = A.n_tiles * BEAM_PARTS;
        const uint2 head = lane < A.segs ? A.heads[row * A.segs + lane] : make_uint2(0, 0);
        float mx = -INFINITY;
        bool bad = false;
        for (int i = lane; i < n_parts; i += WAVE) mx = fmaxf(mx, t[i].mx), bad |= t[i].bad != 0;
        const double c = A.cum[row];
        // ---- what reaches every segment's bound: k logits do
        uint32_t floor = beam_wave_max(head.y);
        // (the lists in registers; of the lanes' largest the k-th, but for its last 6 bits, is a closer bound)
        const int parts = A.list / WAVE;   // of a segment's list
        uint64_t key[BEAM_MAX_ROW_LIST / WAVE];
        uint32_t top = 0;
#pragma unroll
        for (int r = 0; r < BEAM_MAX_ROW_LIST / WAVE; ++r) key[r] = r * WAVE < n_list ? from[r * WAVE + lane] : 0;
#pragma unroll
        for (int r = 0; r < BEAM_MAX_ROW_LIST / WAVE; ++r) {
            const int sg = r / parts, len = r * WAVE < n_list ? __builtin_amdgcn_readlane((int)head.x, sg) : 0;
            if (lane >= len - r % parts * WAVE || (uint32_t)(key[r] >> 32) < floor) key[r] = 0;
            top = max(top, (uint32_t)(key[r] >> 32));
        }
        top = (top & ~63u) | (63 - lane);
        int many = 0;
#pragma unroll
        for (int r = 0; r < BEAM_MAX_ROW_LIST / WAVE; ++r) many += __popcll(__ballot(key[r] != 0));
        if (many > WAVE) floor = max(floor, beam_nth(top, k) & ~63u);
        int n = 0;
#pragma unroll
        for (int r = 0; r < BEAM_MAX_ROW_LIST / WAVE; ++r) {
            if (r * WAVE >= n_list) continue;
            const bool in = key[r] != 0 && (uint32_t)(key[r] >> 32) >= floor;
            const uint64_t m = __ballot(in);
            if (in) mine[n + __popcll(m & ((1ull << lane) - 1))] = key[r];
            n += __popcll(m);
        }
        if (lane < (-n & 7)) mine[n + lane] = 0;   // (read 8 at a time)
        // ---- the row's normaliser
        mx = beam_wave_max(mx);
        const bool dead = __any(bad) || mx == -INFINITY || !(c > -INFINITY);   // uniform over the wave
        double s = 0.0;
        if (!dead)
            for (int i = lane; i < n_parts; i += WAVE) s += t[i].sum * exp((double)t[i].mx - (double)mx);
        s = beam_wave_sum(s);
        const double lse = dead ? 0.0 : (double)mx + log(s);
        // ---- its k largest in order, and their scores (LDS of the wave alone: a fence, and no barrier)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i = lane; i < n && !dead; i += WAVE) {
            const uint64_t key = mine[i];
            int rank = 0;
            for (int j = 0; j < n; j += 8)
#pragma unroll
                for (int e = 0; e < 8; ++e) rank += mine[j + e] > key;
            if (rank < k) {
                rows[b * k + rank] = key;
                score[b * k + rank] = c + ((double)beam_logit(key) - lse);
            }
        }
        if (lane == 0) n_row[b] = dead ? 0 : min(n, k);
    }
    __syncthreads();
    int total = 0;
    for (int b = 0; b < B; ++b) total += n_row[b];
    for (int i = tid; i < B * k; i += BEAM_SEL_THREADS) {
        const int b = i / k, j = i % k;
        if (j >= n_row[b]) continue;
        const double s = score[i];
        int rank = j;
        for (int o = 0; o < B && rank < k; ++o) {
            if (o == b) continue;
            int lo = 0, n = n_row[o];
            while (n > 0) {   // of an earlier beam those with an equal score come first, too
                const int h = n / 2;
                const double x = score[o * k + lo + h];
                if (x > s || (x == s && o < b)) lo += h + 1, n -= h + 1;
                else n = h;
            }
            rank += lo;
        }
        if (rank < k) {
            const int64_t at = (int64_t)p * k + rank;
            A.out_score[at] = s;
            A.out_parent[at] = b;
            A.out_token[at] = beam_token(rows[i]);
        }
    }
    for (int i = total + tid; i < k; i += BEAM_SEL_THREADS) {   // fewer continuations than k
        const int64_t at = (int64_t)p * k + i;
        A.out_score[at] = -INFINITY;
        A.out_parent[at] = -1;
        A.out_token[at] = -1;
    }
}

// Segments per row: enough workgroups for the chip, lists that the second launch holds.
static void beam_plan(BeamArgs& a, int64_t rows) {
    a.n_tiles = (a.vocab + BEAM_TILE - 1) / BEAM_TILE;
    const int64_t want = (2048 + rows - 1) / rows;   // (256 rows of 128256, k 16: 1024 workgroups 55 us, 2048 54, 512 65)
    const int segs = (int)std::min<int64_t>({want, a.n_tiles, BEAM_MAX_ROW_LIST / WAVE, std::max(1, BEAM_MAX_ROW_LIST / (4 * a.k))});
    a.per_seg = (a.n_tiles + segs - 1) / segs;
    a.segs = (a.n_tiles + a.per_seg - 1) / a.per_seg;
    a.list = BEAM_MAX_ROW_LIST / WAVE / a.segs * WAVE;   // whole loads of a wave, 4 k at least (what passes is about 2 k)
}

static int beam_check(int prompts, int beams, int vocab, int k) {
    DKV_REQUIRE(prompts >= 0 && beams > 0, "dkv_beam_select: bad number of prompts or beams");
    DKV_REQUIRE(vocab > 0 && vocab <= 1048576, "dkv_beam_select: vocab must be 1..1048576");
    DKV_REQUIRE(k > 0 && k <= BEAM_MAX_K, "dkv_beam_select: k must be 1..64");
    DKV_REQUIRE((int64_t)beams * k <= BEAM_MAX_LIST, "dkv_beam_select: beams * k must be at most 4096");
    DKV_REQUIRE((int64_t)prompts * beams <= 65535, "dkv_beam_select: more than 65535 rows");
    return DKV_OK;
}

}  // namespace dkv

extern "C" size_t dkv_beam_select_workspace(int32_t prompts, int32_t beams, int32_t vocab, int32_t k) {
    if (dkv::beam_check(prompts, beams, vocab, k) || prompts == 0) return 0;
    dkv::BeamArgs a = {};
    a.vocab = vocab, a.k = k;
    const int64_t rows = (int64_t)prompts * beams;
    dkv::beam_plan(a, rows);
    return rows * (a.n_tiles * dkv::BEAM_PARTS * sizeof(dkv::BeamTile) + (size_t)a.segs * (a.list + 1) * sizeof(uint64_t));
}

extern "C" int dkv_beam_select(const void* logits, int32_t dtype, int64_t row_stride, int32_t prompts, int32_t beams,
                               int32_t vocab, const double* scores, int32_t k, double* out_scores, int32_t* out_parents,
                               int32_t* out_tokens, void* work, size_t work_bytes, dkv_stream_t stream) {
    using namespace dkv;
    if (const int rc = beam_check(prompts, beams, vocab, k)) return rc;
    DKV_REQUIRE(dtype == DKV_F32 || dtype == DKV_BF16, "dkv_beam_select: bad dtype");
    DKV_REQUIRE(row_stride >= vocab, "dkv_beam_select: row_stride is less than vocab");
    if (prompts == 0) return DKV_OK;
    DKV_REQUIRE(logits && scores && out_scores && out_parents && out_tokens, "dkv_beam_select: NULL argument");
    const size_t need = dkv_beam_select_workspace(prompts, beams, vocab, k);
    if (!work || work_bytes < need)
        return fail(DKV_EWORKSPACE, "dkv_beam_select: workspace too small (need " + std::to_string(need) + ")");
    const int64_t rows = (int64_t)prompts * beams;
    BeamArgs a = {};
    a.x = logits, a.cum = scores, a.stride = row_stride, a.vocab = vocab, a.beams = beams, a.k = k;
    beam_plan(a, rows);
    a.tiles = static_cast<BeamTile*>(work);
    a.lists = reinterpret_cast<uint64_t*>(a.tiles + rows * a.n_tiles * BEAM_PARTS);
    a.heads = reinterpret_cast<uint2*>(a.lists + rows * a.segs * a.list);
    a.out_score = out_scores, a.out_parent = out_parents, a.out_token = out_tokens;
    hipStream_t st = as_stream(stream);
    const bool bf = dtype == DKV_BF16;
    // (256 rows of 128256 by vectors and by elements: float32 51 / 52 us, bf16 50 / 54; 32 rows 18 / 19.5)
    const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && row_stride % 4 == 0 && vocab % 4 == 0;
    const dim3 grid(a.segs, (unsigned)rows);
    const auto scan = bf ? (vec ? beam_scan_kernel<true, true> : beam_scan_kernel<true, false>)
                         : (vec ? beam_scan_kernel<false, true> : beam_scan_kernel<false, false>);
    hipLaunchKernelGGL(scan, grid, dim3(BEAM_THREADS), 0, st, a);
    if (const int e = check_launch("dkv_beam_select(scan)")) return e;
    const size_t lds = sizeof(double) * (2 * (size_t)beams * k + (size_t)(BEAM_SEL_THREADS / WAVE) * a.segs * a.list) +
                       sizeof(int) * beams;
    static size_t lds_done[16] = {};
    if (!reserve_lds(reinterpret_cast<const void*>(beam_select_kernel), lds, lds_done))
        return fail(DKV_ELAUNCH, "dkv_beam_select: cannot reserve " + std::to_string(lds) + " B of LDS");
    hipLaunchKernelGGL(beam_select_kernel, dim3(prompts), dim3(BEAM_SEL_THREADS), lds, st, a);
    return check_launch("dkv_beam_select");
}
