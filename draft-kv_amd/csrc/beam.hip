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
//              registers: each tile's maximum and float64 sum of exponentials,
//              and the k largest logits of the segment. The largest of each
//              thread bound the k-th from below, so few logits enter the list
//              that is ranked.
//   2. select  one workgroup per prompt: each row's lse (its tiles in order)
//              and k largest (a rank is a binary search in every segment's
//              sorted list), then the k best of all rows the same way.
// Bound: memory, the logits once; the exponentials (about 20 VALU
// instructions per logit) run beside it.
#include <algorithm>

#include "dexp.h"

namespace dkv {

constexpr int BEAM_THREADS = 256, BEAM_PER = 32;
constexpr int BEAM_TILE = BEAM_THREADS * BEAM_PER;
constexpr int BEAM_MAX_K = 128, BEAM_MAX_LIST = 4096, BEAM_MAX_SEG_LIST = 512;
constexpr int BEAM_SEL_THREADS = 1024;

struct BeamTile {
    double sum;   // of exp(x - mx) over the tile
    float mx;
    int bad;      // the tile holds NaN or +infinity
};

struct BeamArgs {
    const void* x;
    const double* cum;
    int64_t stride;              // elements between rows
    int vocab, beams, k, n_tiles, segs, per_seg;   // tiles per segment
    BeamTile* tiles;             // [row][n_tiles]
    uint64_t* lists;             // [row][segs][k] sorted keys, 0 past the last
    double* out_score;
    int32_t* out_parent;
    int32_t* out_token;
};

// A logit and its index as one number: larger logits first, lower indices first among equal ones.
__device__ __forceinline__ uint64_t beam_key(float x, int i) {
    const uint32_t u = __float_as_uint(x);
    const uint32_t o = (u >> 31) ? ~u : u | 0x80000000u;
    return (uint64_t)o << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float beam_logit(uint64_t key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o >> 31) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int beam_token(uint64_t key) { return (int)~(uint32_t)key; }

// The thread's logits of a tile: element 4 (t + 256 j) + e in register 4 j + e, -infinity past the row. Adding 0 makes
// -0 the 0 that it is equal to.
template <bool BF16, bool VEC>
__device__ __forceinline__ void beam_load(const void* base, int i0, int n, float (&v)[BEAM_PER]) {
#pragma unroll
    for (int j = 0; j < BEAM_PER / 4; ++j) {
        const int i = i0 + 4 * ((int)threadIdx.x + BEAM_THREADS * j);
        if constexpr (VEC) {   // n % 4 == 0: four logits are whole or past the end
            if constexpr (BF16) {
                const uint2 w = i < n ? *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + i)
                                      : make_uint2(0xff80ff80u, 0xff80ff80u);
                v[4 * j] = __uint_as_float(w.x << 16), v[4 * j + 1] = __uint_as_float(w.x & 0xffff0000u);
                v[4 * j + 2] = __uint_as_float(w.y << 16), v[4 * j + 3] = __uint_as_float(w.y & 0xffff0000u);
            } else {
                const float4 w = i < n ? *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i)
                                       : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                v[4 * j] = w.x, v[4 * j + 1] = w.y, v[4 * j + 2] = w.z, v[4 * j + 3] = w.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * j + e] = i + e < n ? load_elem(base, i + e, BF16 ? DKV_BF16 : DKV_F32) : -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < BEAM_PER; ++j) v[j] += 0.0f;
}

// KM: the most k this instance takes
template <bool BF16, bool VEC, int KM>
__global__ void __launch_bounds__(BEAM_THREADS) beam_scan_kernel(BeamArgs A) {
    constexpr int CAP = KM * BEAM_PER + KM;   // at most k threads' logits pass, and the list so far
    __shared__ double tab[EXP_TAB];
    __shared__ uint64_t cand[CAP], best[KM], tmax[BEAM_THREADS];
    __shared__ float wmax[BEAM_THREADS / WAVE];
    __shared__ double wsum[BEAM_THREADS / WAVE];
    __shared__ int n_cand, wbad[BEAM_THREADS / WAVE];
    __shared__ uint64_t s_thr;
    const int seg = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid % WAVE, w = tid / WAVE;
    const int k = A.k;
    const char* base = static_cast<const char*>(A.x) + (int64_t)row * A.stride * (BF16 ? 2 : 4);
    load_exp_tab(tab);
    int n_best = 0;           // uniform
    uint64_t kth = 0;         // the k-th best so far (0: fewer than k)
    const int t0 = seg * A.per_seg, t1 = min(t0 + A.per_seg, A.n_tiles);
    for (int tile = t0; tile < t1; ++tile) {
        const int i0 = tile * BEAM_TILE;
        float v[BEAM_PER];
        beam_load<BF16, VEC>(base, i0, A.vocab, v);
        // ---- the thread's largest, the first of them
        float mx = -INFINITY;
        int arg = 0;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < BEAM_PER; ++j) {
            bad |= !(v[j] < INFINITY);
            if (v[j] > mx) mx = v[j], arg = j;   // (indices rise with j)
        }
        const int at = i0 + 4 * (tid + BEAM_THREADS * (arg / 4)) + arg % 4;
        const uint64_t mine = mx > -INFINITY ? beam_key(mx, at) : 0;
        tmax[tid] = mine;
        const float wm = wave_max(mx);
        const uint64_t wb = __ballot(bad);
        if (lane == 0) wmax[w] = wm, wbad[w] = wb != 0;
        if (tid == 0) n_cand = 0, s_thr = 0;
        __syncthreads();
        float tm = wmax[0];
        bool tbad = false;
#pragma unroll
        for (int i = 0; i < BEAM_THREADS / WAVE; ++i) tm = fmaxf(tm, wmax[i]), tbad |= wbad[i] != 0;
        // ---- what a candidate must reach: the k-th largest of the threads' largest, or the k-th so far
        if (mine > kth) {
            int rank = 0;
            for (int i = 0; i < BEAM_THREADS; ++i) rank += tmax[i] > mine;
            if (rank == k - 1) s_thr = mine;
        }
        // ---- exponentials
        const double m = tm == -INFINITY ? 0.0 : (double)tm;
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < BEAM_PER; j += 8) {
            double y[8], ex[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (double)v[j + e] - m;
            dexp_n<8>(y, ex, tab);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += ex[e];
        }
        sum = wave_sum_d(sum);
        if (lane == 0) wsum[w] = sum;
        __syncthreads();
        if (tid == 0) {
            double s = 0.0;
            for (int i = 0; i < BEAM_THREADS / WAVE; ++i) s += wsum[i];
            A.tiles[(int64_t)row * A.n_tiles + tile] = BeamTile{s, tm, tbad};
        }
        const uint64_t thr = s_thr > kth ? s_thr : kth;
        const float thr_x = thr ? beam_logit(thr) : -INFINITY;
        if (mine > kth && mx >= thr_x) {
#pragma unroll
            for (int j = 0; j < BEAM_PER; ++j)
                if (v[j] >= thr_x && v[j] > -INFINITY) {
                    const uint64_t key = beam_key(v[j], i0 + 4 * (tid + BEAM_THREADS * (j / 4)) + j % 4);
                    // (the threshold itself is one of the candidates; the k-th so far is in the list)
                    if (key > kth && key >= thr) cand[atomicAdd(&n_cand, 1)] = key;
                }
        }
        __syncthreads();
        int n = n_cand;
        if (n > 0) {   // uniform
            if (tid < n_best) cand[n + tid] = best[tid];
            __syncthreads();
            n += n_best;
            for (int i = tid; i < n; i += BEAM_THREADS) {
                const uint64_t key = cand[i];
                int rank = 0;
                for (int j = 0; j < n; ++j) rank += cand[j] > key;
                if (rank < k) best[rank] = key;
            }
            n_best = min(n, k);
            __syncthreads();
            kth = n_best == k ? best[k - 1] : 0;
        }
    }
    uint64_t* out = A.lists + ((int64_t)row * A.segs + seg) * k;
    for (int i = tid; i < k; i += BEAM_THREADS) out[i] = i < n_best ? best[i] : 0;
}

// How many of the sorted keys a[0 .. n) are larger than key
__device__ __forceinline__ int beam_above(const uint64_t* a, int n, uint64_t key) {
    int lo = 0;
    while (n > 0) {
        const int h = n / 2;
        if (a[lo + h] > key) lo += h + 1, n -= h + 1;
        else n = h;
    }
    return lo;
}

__global__ void __launch_bounds__(BEAM_SEL_THREADS) beam_select_kernel(BeamArgs A) {
    extern __shared__ __align__(16) char lds[];
    const int B = A.beams, k = A.k, n_list = A.segs * k;
    constexpr int NW = BEAM_SEL_THREADS / WAVE;
    double* tab = reinterpret_cast<double*>(lds);
    double* cum = tab + EXP_TAB;                               // [B]
    double* lse = cum + B;                                     // [B]
    uint64_t* rows = reinterpret_cast<uint64_t*>(lse + B);     // [B][k]
    uint64_t* seg = rows + B * k;                              // [NW][segs * k]
    int* n_row = reinterpret_cast<int*>(seg + NW * n_list);    // [B] live candidates of a row
    const int p = blockIdx.x, tid = threadIdx.x, lane = tid % WAVE, w = tid / WAVE;
    load_exp_tab(tab);
    __syncthreads();
    for (int b = w; b < B; b += NW) {
        const int64_t row = (int64_t)p * B + b;
        uint64_t* mine = seg + w * n_list;
        for (int i = lane; i < n_list; i += WAVE) mine[i] = A.lists[row * n_list + i];
        for (int i = lane; i < k; i += WAVE) rows[b * k + i] = 0;
        // ---- the row's normaliser
        const BeamTile* t = A.tiles + row * A.n_tiles;
        float mx = -INFINITY;
        bool bad = false;
        for (int i = lane; i < A.n_tiles; i += WAVE) mx = fmaxf(mx, t[i].mx), bad |= t[i].bad != 0;
        mx = wave_max(mx);
        const double c = A.cum[row];
        const bool dead = __any(bad) || mx == -INFINITY || !(c > -INFINITY);   // uniform over the wave
        double s = 0.0;
        if (!dead)
            for (int i = lane; i < A.n_tiles; i += WAVE) s += t[i].sum * dexp((double)t[i].mx - (double)mx, tab);
        s = wave_sum_d(s);
        if (lane == 0) {
            cum[b] = c;
            lse[b] = dead ? 0.0 : (double)mx + log(s);
        }
        // ---- its k largest (LDS of the wave alone: a fence, and no barrier)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        int live = 0;
        for (int i = lane; i < n_list; i += WAVE) {
            const uint64_t key = dead ? 0 : mine[i];
            if (key == 0) continue;
            int rank = 0;
            for (int g = 0; g < A.segs; ++g) rank += beam_above(mine + g * k, k, key);
            if (rank < k) rows[b * k + rank] = key, ++live;
        }
        live = wave_sum_i(live);
        if (lane == 0) n_row[b] = live;
    }
    __syncthreads();
    auto score = [&](int b, int j) { return cum[b] + ((double)beam_logit(rows[b * k + j]) - lse[b]); };
    int total = 0;
    for (int b = 0; b < B; ++b) total += n_row[b];
    for (int i = tid; i < B * k; i += BEAM_SEL_THREADS) {
        const int b = i / k, j = i % k;
        if (j >= n_row[b]) continue;
        const double s = score(b, j);
        int rank = j;
        for (int o = 0; o < B && rank < k; ++o) {
            if (o == b) continue;
            int lo = 0, n = n_row[o];
            while (n > 0) {   // of an earlier beam those with an equal score come first, too
                const int h = n / 2;
                const double x = score(o, lo + h);
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
    const int64_t want = (1024 + rows - 1) / rows;
    const int segs = (int)std::min<int64_t>({want, a.n_tiles, std::max(1, BEAM_MAX_SEG_LIST / a.k)});
    a.per_seg = (a.n_tiles + segs - 1) / segs;
    a.segs = (a.n_tiles + a.per_seg - 1) / a.per_seg;
}

static int beam_check(int prompts, int beams, int vocab, int k) {
    DKV_REQUIRE(prompts >= 0 && beams > 0, "dkv_beam_select: bad number of prompts or beams");
    DKV_REQUIRE(vocab > 0 && vocab <= 1048576, "dkv_beam_select: vocab must be 1..1048576");
    DKV_REQUIRE(k > 0 && k <= BEAM_MAX_K, "dkv_beam_select: k must be 1..128");
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
    return rows * (a.n_tiles * sizeof(dkv::BeamTile) + (size_t)a.segs * k * sizeof(uint64_t));
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
    a.lists = reinterpret_cast<uint64_t*>(a.tiles + rows * a.n_tiles);
    a.out_score = out_scores, a.out_parent = out_parents, a.out_token = out_tokens;
    hipStream_t st = as_stream(stream);
    const bool bf = dtype == DKV_BF16;
    const bool vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && row_stride % 4 == 0 && vocab % 4 == 0;
    const dim3 grid(a.segs, (unsigned)rows);
#define DKV_SCAN(BB, VV)                                                                                                    \
    do {                                                                                                                    \
        if (k <= 32) hipLaunchKernelGGL((beam_scan_kernel<BB, VV, 32>), grid, dim3(BEAM_THREADS), 0, st, a);                \
        else hipLaunchKernelGGL((beam_scan_kernel<BB, VV, BEAM_MAX_K>), grid, dim3(BEAM_THREADS), 0, st, a);                \
    } while (0)
    if (bf && vec) DKV_SCAN(true, true);
    else if (bf) DKV_SCAN(true, false);
    else if (vec) DKV_SCAN(false, true);
    else DKV_SCAN(false, false);
#undef DKV_SCAN
    if (const int e = check_launch("dkv_beam_select(scan)")) return e;
    const size_t lds = sizeof(double) * (EXP_TAB + 2 * beams) +
                       sizeof(uint64_t) * ((size_t)beams * k + (size_t)(BEAM_SEL_THREADS / WAVE) * a.segs * k) + sizeof(int) * beams;
    static size_t lds_done[16] = {};
    if (!reserve_lds(reinterpret_cast<const void*>(beam_select_kernel), lds, lds_done))
        return fail(DKV_ELAUNCH, "dkv_beam_select: cannot reserve " + std::to_string(lds) + " B of LDS");
    hipLaunchKernelGGL(beam_select_kernel, dim3(prompts), dim3(BEAM_SEL_THREADS), lds, st, a);
    return check_launch("dkv_beam_select");
}
