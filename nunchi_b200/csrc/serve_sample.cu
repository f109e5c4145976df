// Sampling a word per row of scores (imi_cuda_sample): temperature, top-k, top-p and min-p, from a given uniform number.
//
// With w_j = exp((x_j - max x) / temperature) the three filters keep a prefix of the words ordered by (score, id): the
// first k; those before which less than p of the mass lies; those of w >= m. So the kept set is "score above a value T,
// and the first c of the words at T", and the pick is the first word, by id, at which the running kept mass exceeds
// u times its total. Weights are held as integers of 2^-44 (1 is the largest word's): sums are exact whatever the order
// they are made in, so atomics and parallel sums cannot change which word a border falls on, and 2^18 words fit 62 bits.
// exp and the borders are computed in 64 bits: a border is missed only where two candidates differ by about 2^-44.
//
// A row is held in the shared memory of a cluster of 1 to 8 CTAs, as integer keys that order like the scores: it is
// read from HBM once, and every later pass is over shared memory.
//   The list: while loading, every thread keeps its own words' maximum. The r-th largest of a CTA's thread maxima is a value
// that r of its words reach, so the smallest of these over the cluster, with r = ceil(k / CTAs), is one that k words reach;
// for top-p alone r is set for about 500 words, for min-p alone the value follows from the maximum. The words above it are
// listed, and one CTA applies the filters to the list. What top-p needs of the other words is their mass: it is summed
// in 32 bits, and only where the nucleus's end depends on the error of that sum, or lies below the list, in full.
//   A nucleus, or a top-k, that goes on below the list: a histogram over 1,024 steps of score, of masses (or counts), is
// searched, the crossing bin's words listed and searched in turn; a bin too full for a list (scores crowded in few steps,
// masked words) is cut again, by keys, until it fits or is a single value. Then every CTA sums its kept words by id.
// Measured on rows of 97,496: one by top-k 50 and top-p 8.0 us; 64 by top-k 50 and top-p 12.4, by top-p 0.9 alone 51 (7 rows below
// the list; the others are done at 14); 256 of bf16 with mixed settings 76. Bound by the chains of barriers and searches.
#include "common.cuh"
#include "serve.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace imi {
namespace {

constexpr int SM_NT = 32 * SM_NW;
constexpr int SM_BINS = 2 * SM_NT;       // two bins per thread in the scans
constexpr int SM_SHORT = SM_NT / 4;      // words of a list that are all compared with one another
constexpr int SM_PILES = 256;            // piles that a search in a longer list throws its words into
constexpr int SM_STEPS = 256;            // steps in which the threads' maxima are ranked
// the 32-bit mass's relative error at most: of a word's exponent (up to 45) 2^-23 twice, in powers of 2, its exp2 2^-22, the
// sum of up to 64 words of a thread 2^-18; the threads' sums are added in 64 bits
constexpr double SM_MASS_ERR = 45 * 0.7 * 2.4e-7 + 2.4e-7 + 3.9e-6;
constexpr double SM_ONE = 17592186044416.0;   // 2^44
static_assert((long long) SM_SLICE * SM_MAX_CLUSTER >= IMI_CUDA_SAMPLE_VOCAB, "a row fits a cluster");
static_assert((long long) IMI_CUDA_SAMPLE_VOCAB <= 1 << 18, "the weights' sum fits 62 bits");

typedef unsigned long long u64;

struct SampleArgs {
    imi_cuda_sample_args a;
    int seg, share, rank;      // sample_split
    const void *const *rows;   // the rows' scores where they do not lie `stride` apart (the engine's conversations)
    SessDev *const *states;    // and the conversations whose last pick each row's word becomes (not if there is none)
};

// scores as unsigned keys in the same order; NaN is -infinity, whose key no kept word has; the zeros are one
constexpr uint32_t KEY_NONE = 0x007FFFFFu;
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(__fadd_rn(fmaxf(x, -INFINITY), 0.0f));
    return b ^ ((uint32_t) ((int) b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

struct SampleShared {
    union {
        struct {
            unsigned bins[3][SM_BINS];   // this CTA's histogram: words, or their masses' 15-bit digits (2^15 words at most)
        };
        struct {
            u64 list[SM_LIST];               // leading CTA: (key, ~id) of all CTAs' words
            u64 w[SM_LIST];                  // this CTA's words until they are there; then the list's weights
            unsigned pile[SM_PILES][2];      // masses, low and high words
            unsigned short member[SM_LIST];
        };
        struct {
            u64 list_[SM_LIST];
            unsigned steps[SM_STEPS];        // the threads' maxima ranked
        };
        unsigned queue[SM_NW][64];           // the warps' kept words
    };
    unsigned wc[SM_NW];               // scans over the CTA
    u64 wm[SM_NW];
    double2 near[SM_NW];
    // what the cluster reads of this CTA
    unsigned mx, mn, lmin, nvalid, floor, idmin, n_list, n_all, at_lead, part_kept, lo, hi;
    // of every CTA of the cluster, written here by it: read after a barrier, and never by two exchanges in a row
    unsigned all_mx[SM_MAX_CLUSTER], all_floor[SM_MAX_CLUSTER], all_n[SM_MAX_CLUSTER], all_cnt[SM_MAX_CLUSTER], all_kept[SM_MAX_CLUSTER];
    double all_near[SM_MAX_CLUSTER], all_listed[SM_MAX_CLUSTER];
    u64 all_mass[SM_MAX_CLUSTER], all_sum[SM_MAX_CLUSTER];
    u64 mass_above;
    int bin;                          // found in a scan: the crossing bin, and what lies above it
    unsigned above;
    unsigned T, c, done;              // the leading CTA's findings
    u64 found, found_after;           // a search in the list
    u64 total;
    unsigned n_member;
};

// exclusive sums over the CTA's threads, and the totals
__device__ __forceinline__ void scan2(SampleShared &s, unsigned &c, u64 &m, unsigned &tc, u64 &tm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned xc = c;
    u64 xm = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned yc = __shfl_up_sync(~0u, xc, o);
        const u64 ym = __shfl_up_sync(~0u, xm, o);
        if (lane >= o) { xc += yc; xm += ym; }
    }
    __syncthreads();
    if (lane == 31) { s.wc[warp] = xc; s.wm[warp] = xm; }
    __syncthreads();
    unsigned bc = 0;
    u64 bm = 0;
    tc = 0;
    tm = 0;
#pragma unroll
    for (int w = 0; w < SM_NW; w++) {
        if (w < warp) { bc += s.wc[w]; bm += s.wm[w]; }
        tc += s.wc[w];
        tm += s.wm[w];
    }
    c = bc + xc - c;
    m = bm + xm - m;
}

// A word's weight, as a number and as an integer of 2^-44. With y = -z log2 e and n the nearest integer to it, exp(-z) = 2^n 2^r,
// |r| <= 1/2; 2^r by the polynomial through its values at 11 Chebyshev nodes (relative error below 2^-51). A table and a
// shorter polynomial took twice as long: 32 lanes' reads of it fall on a few banks. What bounds a pass of this over a row is the
// 15 operations in 64 bits (61 a nanosecond and SM: 6 of the 11.5 us that a CTA's 24,400 words take; their histogram hides behind).
struct Weigher {
    double xmax, c;    // the largest score; log2(e) / temperature
    float low;         // scores further down than this weigh 0; they are raised to it
    uint32_t kmax;
    bool odd;          // an infinite largest score, temperatures out of all proportion, a min-p below the weights' resolution
    __device__ __forceinline__ double real(float x) const {   // no branches: several words are in flight at once
        constexpr double MAGIC = 6755399441055744.0;   // 1.5 * 2^52: adding it leaves the nearest integer in the low bits
        const double d = (double) fmaxf(x, low) - xmax, b = __fma_rn(d, c, MAGIC);
        const double r = __fma_rn(d, c, -__dadd_rn(b, -MAGIC));
        double e = __fma_rn(r, 7.072585949269224e-09, 1.0208690299958306e-07);
        e = __fma_rn(r, e, 1.321544258792169e-06);
        e = __fma_rn(r, e, 1.5252657260200837e-05);
        e = __fma_rn(r, e, 0.0001540353044173605);
        e = __fma_rn(r, e, 0.0013333558230164974);
        e = __fma_rn(r, e, 0.009618129107606888);
        e = __fma_rn(r, e, 0.05550410866444772);
        e = __fma_rn(r, e, 0.24022650695910097);
        e = __fma_rn(r, e, 0.69314718055995);
        e = __fma_rn(r, e, 1.0);
        return __hiloint2double(__double2hiint(e) + __double2loint(b) * (1 << 20), __double2loint(e));
    }
    __device__ __noinline__ double rare(uint32_t k) const {
        if (k == kmax) return 1.0;
        const double z = (xmax - (double) value_of(k)) * (c * 0.69314718055994530942);
        return k > KEY_NONE && z >= 0.0 ? exp(-z) : 0.0;   // z NaN: below an infinite score
    }
    __device__ __forceinline__ double real(uint32_t k) const { return odd ? rare(k) : real(value_of(k)); }
    // w * 2^44 <= 2^44: added to 2^52 its integer part, rounded to nearest, is the low mantissa. raw: with the exponent's bits
    // still in place, which sums of n words hold n times (as 64 bits go)
    static constexpr u64 RAW = 0x4330000000000000ull;
    static __device__ __forceinline__ u64 raw(double w) { return (u64) __double_as_longlong(__fma_rn(w, SM_ONE, 4503599627370496.0)); }
    static __device__ __forceinline__ u64 whole(double w) { return raw(w) - RAW; }
    __device__ __forceinline__ u64 operator()(uint32_t k) const { return whole(real(k)); }
    // four words' at once, with one branch for all: their chains of operations go side by side
    __device__ __forceinline__ void four(const uint4 &q, double (&w)[4]) const {
        if (odd) {
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = rare((&q.x)[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = real(value_of((&q.x)[e]));
        }
    }
    __device__ __forceinline__ u64 raw4(const uint4 &q) const {
        double w[4];
        four(q, w);
        return (raw(w[0]) + raw(w[1])) + (raw(w[2]) + raw(w[3]));
    }
    __device__ __forceinline__ float logprob(uint32_t k, u64 total) const {
        const double d = k == kmax ? 0.0 : ((double) value_of(k) - xmax) * c * 0.69314718055994530942;
        return (float) (d - log((double) total / SM_ONE));
    }
};

// 64-bit addition by halves: the carry is what the low half's old value shows
__device__ __forceinline__ void add64(unsigned (&at)[2], u64 w) {
    const unsigned wl = (unsigned) w, old = atomicAdd(&at[0], wl), wh = (unsigned) (w >> 32) + (old + wl < old);
    if (wh) atomicAdd(&at[1], wh);
}
// A search in the list of n words: in the order of ord (larger first; no two alike), the word with cross(b, b + weight) where
// b is what lies before it, `above` more than the words in front of it in the list. pile(word) is 0..SM_PILES-1 in that order,
// or -1 for a word that is not in question. The piles' sums show which pile it is in, a comparison of that pile's words which it
// is: no sort. s.found is 0 if there is none; s.found_after is the sum up to and with it.
template <typename P, typename W, typename O, typename X>
__device__ __forceinline__ void search_list(SampleShared &s, int n, u64 above, P pile, W weight, O ord, X cross) {
    const int tid = threadIdx.x, lane = tid & 31;
    for (int i = tid; i < SM_PILES; i += SM_NT) s.pile[i][0] = s.pile[i][1] = 0;
    if (tid == 0) { s.found = s.found_after = 0; s.n_member = 0; }
    __syncthreads();
    for (int i = tid; i < n; i += SM_NT) {
        const int b = pile(s.list[i]);
        if (b >= 0) add64(s.pile[b], weight(i));
    }
    __syncthreads();
    u64 v[SM_PILES / 32], sum = 0;
#pragma unroll
    for (int e = 0; e < SM_PILES / 32; e++) {
        const unsigned *q = s.pile[SM_PILES / 32 * lane + e];
        sum += v[e] = (u64) q[1] << 32 | q[0];
    }
    u64 b = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(~0u, b, o);
        if (lane >= o) b += y;
    }
    b += above - sum;
    int at = -1;
    u64 before = 0;
#pragma unroll
    for (int e = 0; e < SM_PILES / 32; e++) {
        if (at < 0 && cross(b, b + v[e])) { at = SM_PILES / 32 * lane + e; before = b; }
        b += v[e];
    }
    const unsigned who = __ballot_sync(~0u, at >= 0);
    if (!who) return;   // the same for every warp
    at = __shfl_sync(~0u, at, __ffs(who) - 1);
    before = __shfl_sync(~0u, before, __ffs(who) - 1);
    for (int i = tid; i < n; i += SM_NT)
        if (pile(s.list[i]) == at) s.member[atomicAdd(&s.n_member, 1u)] = (unsigned short) i;
    __syncthreads();
    const int m = (int) s.n_member;
    for (int i = tid; i < m; i += SM_NT) {
        const int j0 = s.member[i];
        const auto mine = ord(s.list[j0]);
        u64 x = before;
        for (int k = 0; k < m; k++) {
            const int j = s.member[k];
            if (ord(s.list[j]) > mine) x += weight(j);
        }
        const u64 y = x + weight(j0);
        if (cross(x, y)) { s.found = s.list[j0]; s.found_after = y; }
    }
    __syncthreads();
}

template <typename S>
__device__ __forceinline__ float score_at(const S *x, int i) {
    if constexpr (sizeof(S) == 4) return x[i];
    else if constexpr (std::is_same<S, __half>::value) return __half2float(x[i]);
    else return __bfloat162float(x[i]);
}

template <typename S> struct Four { typedef uint2 T; };   // four scores
template <> struct Four<float> { typedef uint4 T; };

// a value of every CTA of the cluster: lane r holds CTA r's (other lanes `none`), read at once
#define OF_CTAS(field, none) (lane < C ? cl.map_shared_rank(&s, lane)->field : (none))
template <typename V>
__device__ __forceinline__ V sum8(V v) {   // over the first 8 lanes, to all
#pragma unroll
    for (int o = 4; o; o >>= 1) v += __shfl_down_sync(~0u, v, o);
    return __shfl_sync(~0u, v, 0);
}

template <typename S>
__global__ void __launch_bounds__(SM_NT, 2) k_sample(const __grid_constant__ SampleArgs p) {
    extern __shared__ __align__(16) uint8_t sm_raw[];
    SampleShared &s = *(SampleShared *) sm_raw;
    uint32_t *keys = (uint32_t *) (sm_raw + (sizeof(SampleShared) + 15) / 16 * 16);
    const imi_cuda_sample_args &a = p.a;
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int) cl.num_blocks(), rank = (int) cl.block_rank();
    const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int base = rank * p.share, end = min(a.vocab, base + p.share);   // this CTA's words
    if (tid == 0) { s.mx = 0; s.mn = ~0u; s.nvalid = 0; s.idmin = ~0u; s.n_list = s.n_all = 0; s.floor = s.lmin = ~0u; }
    if (tid < SM_STEPS) s.steps[tid] = 0;
    __syncthreads();
    auto started = cl.barrier_arrive();   // this CTA's shared memory may be written by the others
    pdl_wait();
    pdl_trigger();
    const float temp = a.temperature ? a.temperature[row] : 1.0f, top_p = a.top_p ? a.top_p[row] : 1.0f,
                min_p = a.min_p ? a.min_p[row] : 0.0f;
    int top_k = a.top_k ? a.top_k[row] : 0;
    float u = a.u[row];
    u = u >= 0.0f ? fminf(u, 0.99999994f) : 0.0f;          // NaN: 0
    const bool greedy = !(temp > 0.0f);
    if (top_p <= 0.0f) top_k = 1;                           // the first word alone
    const bool use_k = top_k > 0 && top_k < a.vocab, use_p = top_p > 0.0f && top_p < 1.0f, use_m = min_p > 0.0f;
    const double m = fmin((double) min_p, 1.0), pd = (double) top_p;

    // the row as keys; the largest
    const S *x = p.rows ? (const S *) p.rows[row] : (const S *) a.scores + row * a.stride;
    const bool vec = ((uintptr_t) (x + base) & (4 * sizeof(S) - 1)) == 0;
    uint32_t mx = 0;
    uint32_t *mine = keys + warp * p.seg + 4 * lane;        // the words of a lane, tile by tile
    const int first = base + warp * p.seg + 4 * lane;
    auto put = [&](int o, const float (&f)[4]) {
        uint4 k = make_uint4(key_of(f[0]), key_of(f[1]), key_of(f[2]), key_of(f[3]));
        mx = max(max(mx, max(k.x, k.y)), max(k.z, k.w));
        *(uint4 *) (mine + o) = k;
    };
    const int inside = end - (base + warp * p.seg);         // words of the row in this warp's part
    const int whole = vec ? max(0, min(p.seg, inside / SM_TILE * SM_TILE)) : 0;
    int o = 0;
    constexpr int BATCH = sizeof(S) == 4 ? 4 : 6;           // tiles' loads in flight
    for (; o + BATCH * SM_TILE <= whole; o += BATCH * SM_TILE) {
        typename Four<S>::T v[BATCH];
#pragma unroll
        for (int t = 0; t < BATCH; t++) v[t] = __ldg((const typename Four<S>::T *) (x + first + o + t * SM_TILE));
#pragma unroll
        for (int t = 0; t < BATCH; t++) {
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = score_at((const S *) &v[t], e);
            put(o + t * SM_TILE, f);
        }
    }
    for (; o < p.seg; o += SM_TILE) {
        float f[4];
        if (o < whole) {
            const typename Four<S>::T v = __ldg((const typename Four<S>::T *) (x + first + o));
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = score_at((const S *) &v, e);
        } else
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = first + o + e < end ? score_at(x, first + o + e) : -INFINITY;
        put(o, f);
    }
    // the value that the r-th largest of the threads' maxima reaches: the maxima ranked in 256 steps, all steps down to the
    // one of the r-th taken whole
    const bool by_k = use_k && top_k <= SM_LIST, by_p = !use_k && use_p, by_m = !use_k && !use_p && use_m;
    const int r_th = by_k ? (top_k + C - 1) / C : by_p ? p.rank : 0;
    const bool lists = !greedy && r_th <= SM_NT && (by_k || by_p || by_m);
    const uint32_t lmx = mx, wmax = __reduce_max_sync(~0u, mx);
    if (lane == 0) atomicMax(&s.mx, wmax);
    if (lists && r_th) {
        const uint32_t wmin = __reduce_min_sync(~0u, mx > KEY_NONE ? mx : ~0u);
        if (lane == 0) atomicMin(&s.lmin, wmin);
        __syncthreads();
        // masked words of low values must not stretch the steps: what lies further down shares the last one
        const float top = value_of(s.mx), span = fminf(__fadd_rn(top, -value_of(min(s.lmin, s.mx))), 64.0f);
        const float sc = span > 0.0f ? __fdiv_rn((float) SM_STEPS, span) : 0.0f;
        const int st = lmx <= KEY_NONE || lmx == s.mx ? (lmx <= KEY_NONE ? SM_STEPS - 1 : 0)
                                                      : min(SM_STEPS - 1, __float2int_rz(__fmul_rn(__fadd_rn(top, -value_of(lmx)), sc)));
        unsigned *h = s.steps;
        atomicAdd(&h[st], 1u);
        __syncthreads();
        unsigned c8[8], c = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) c += c8[e] = h[8 * lane + e];
        unsigned up = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(~0u, up, o);
            if (lane >= o) up += y;
        }
        int step = SM_STEPS;
        unsigned run = up - c;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (run < (unsigned) r_th && run + c8[e] >= (unsigned) r_th) step = 8 * lane + e;
            run += c8[e];
        }
        step = __reduce_min_sync(~0u, step);
        const uint32_t low = __reduce_min_sync(~0u, st <= step ? lmx : ~0u);
        if (lane == 0) atomicMin(&s.floor, low);
    }
    __syncthreads();
    cl.barrier_wait(std::move(started));
    if (tid < C) {
        SampleShared &o = *cl.map_shared_rank(&s, tid);
        o.all_mx[rank] = s.mx;
        o.all_floor[rank] = s.floor;
    }
    cl.sync();
    mx = __reduce_max_sync(~0u, lane < C ? s.all_mx[lane] : 0u);
    uint32_t floor = max(__reduce_min_sync(~0u, lane < C ? s.all_floor[lane] : ~0u), KEY_NONE + 1);
    auto emit = [&](int id, float lp, int kept) {
        a.ids[row] = id;
        if (p.states && id >= 0) {
            p.states[row]->next_token = id;
            p.states[row]->amax_val = score_at(x, id);
        }
        if (a.logprob) a.logprob[row] = lp;
        if (a.kept) a.kept[row] = kept;
    };
    if (mx <= KEY_NONE) {
        if (rank == 0 && tid == 0) emit(-1, -INFINITY, 0);
        return;
    }
    const float xmax = value_of(mx);
    if (greedy) {
        unsigned id = ~0u;
        if (wmax == mx)
            for (int o = 0; o < p.seg; o += SM_TILE)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (mine[o + e] == mx) id = min(id, (unsigned) (first + o + e));
        id = __reduce_min_sync(~0u, id);
        if (lane == 0 && id != ~0u) atomicMin(&cl.map_shared_rank(&s, 0)->idmin, id);
        cl.sync();
        if (rank == 0 && tid == 0) emit((int) s.idmin, 0.0f, 1);
        return;
    }
    // 32.5 temperatures down a weight is below 2^-46, and rounds to 0
    const Weigher weigh = { (double) xmax, 1.4426950408889634074 / (double) temp, __fmaf_rn(-32.5f, temp, xmax), mx,
                            !(temp >= fabsf(xmax) * 0x1p-16f && temp > 1e-30f && temp < 1e30f) || (use_m && m < 1e-12) };

    // searches in the leading CTA's list
    constexpr u64 PASS = 1ull << 63;   // with a weight: the word passes min-p
    auto weigh_list = [&](int n) {
        for (int i = tid; i < n; i += SM_NT) {
            const double w = weigh.real((uint32_t) (s.list[i] >> 32));
            s.w[i] = Weigher::whole(w) | (!use_m || w >= m ? PASS : 0);
        }
    };
    // the smallest and the largest of f(word) over the list
    auto ends = [&](int n, auto f, uint32_t &lo, uint32_t &hi) {
        uint32_t l = ~0u, h = 0;
        for (int i = tid; i < n; i += SM_NT) {
            const uint32_t v = f(s.list[i]);
            l = min(l, v);
            h = max(h, v);
        }
        l = __reduce_min_sync(~0u, l);
        h = __reduce_max_sync(~0u, h);
        __syncthreads();
        if (lane == 0) s.wm[warp] = (u64) l << 32 | h;
        __syncthreads();
        const u64 v = s.wm[lane % SM_NW];
        lo = __reduce_min_sync(~0u, (unsigned) (v >> 32));
        hi = __reduce_max_sync(~0u, (unsigned) v);
    };
    auto by_score = [&](int n, u64 above, auto weight, auto cross) {
        uint32_t lo, hi;
        ends(n, [](u64 q) { return (uint32_t) (q >> 32); }, lo, hi);
        const float top = value_of(hi), sp = fminf(__fadd_rn(top, -value_of(lo)), 3e38f), f = sp > 0.0f ? __fdiv_rn((float) SM_PILES, sp) : 0.0f;
        search_list(s, n, above, [&](u64 q) -> int {
            const uint32_t k = (uint32_t) (q >> 32);
            return k == hi ? 0 : min(SM_PILES - 1, __float2int_rz(__fmul_rn(__fadd_rn(top, -value_of(k)), f)));
        }, weight, [](u64 q) { return q; }, cross);
    };
    auto whole_of = [&](int i) -> u64 { return s.w[i] & ~PASS; };
    // what the list's words from `last` on upwards weigh together
    auto list_mass = [&](int n, u64 last, bool pass, unsigned &cnt) -> u64 {
        u64 sum = 0, total;
        unsigned c = 0;
        for (int i = tid; i < n; i += SM_NT)
            if (s.list[i] >= last && (!pass || (s.w[i] & PASS))) { sum += s.w[i] & ~PASS; c++; }
        scan2(s, c, sum, cnt, total);
        return total;
    };
    // a short list: four threads per word compare it with all others. The word's place in the order of scores, the mass before
    // it and with it (all four threads)
    struct Place {
        bool in;
        int rank;
        u64 before, after;
    };
    auto quad = [&](u64 v) {
        v += __shfl_xor_sync(~0u, v, 1);
        return v + __shfl_xor_sync(~0u, v, 2);
    };
    auto place = [&](int n) -> Place {
        Place r = { tid / 4 < n, 0, 0, 0 };
        if (r.in) {
            const u64 q = s.list[tid / 4];
#pragma unroll 4
            for (int j = tid & 3; j < n; j += 4)
                if (s.list[j] > q) { r.rank++; r.before += s.w[j] & ~PASS; }
        }
        r.rank += __shfl_xor_sync(~0u, r.rank, 1);
        r.rank += __shfl_xor_sync(~0u, r.rank, 2);
        r.before = quad(r.before);
        r.after = r.in ? r.before + (s.w[tid / 4] & ~PASS) : 0;
        return r;
    };
    auto short_pick = [&](int n, bool keep) {
        const int i = tid / 4;
        keep = keep && (s.w[i] & PASS);
        const u64 w = keep ? s.w[i] & ~PASS : 0, q = i < n ? s.list[i] : 0;
        __syncthreads();
        if ((tid & 3) == 0 && i < n) s.w[i] = w;
        const int K = __syncthreads_count(keep) / 4;
        u64 b = 0, t = 0;
#pragma unroll 4
        for (int j = tid & 3; j < n; j += 4) {
            const u64 wj = s.w[j];
            t += wj;
            if ((unsigned) s.list[j] > (unsigned) q) b += wj;   // ~id larger: id smaller
        }
        b = quad(b);
        t = quad(t);
        const double target = (double) u * (double) t;
        if ((tid & 3) == 0 && keep && (double) b <= target && (double) (b + w) > target)
            emit((int) ~(unsigned) q, weigh.logprob((uint32_t) (q >> 32), t), K);
    };
    // the pick, by id, among the list's words from `last` on upwards that pass min-p
    auto pick = [&](int n, u64 last) {
        unsigned K;
        const u64 total = list_mass(n, last, true, K);
        const double target = (double) u * (double) total;
        uint32_t lo, hi;   // of ~id: larger first
        ends(n, [](u64 q) { return (uint32_t) q; }, lo, hi);
        const float f = __fdiv_rn((float) SM_PILES, (float) (hi - lo + 1));
        search_list(s, n, 0, [&](u64 q) -> int { return min(SM_PILES - 1, (int) __fmul_rn((float) (hi - (unsigned) q), f)); }, [&](int i) -> u64 { return s.list[i] >= last && (s.w[i] & PASS) ? s.w[i] & ~PASS : 0; },
            [](u64 q) { return (unsigned) q; }, [&](u64 b, u64 e) { return (double) b <= target && (double) e > target; });
        if (tid == 0) emit((int) ~(unsigned) s.found, weigh.logprob((uint32_t) (s.found >> 32), total), (int) K);
    };

    // this CTA's words to the leading one's list, behind those that came before, and its count to every CTA (too many words are
    // cut: the counts show it). A cluster barrier comes next
    auto push_list = [&]() {
        __syncthreads();
        SampleShared &lead = *cl.map_shared_rank(&s, 0);
        const unsigned n = s.n_list;
        if (tid == 0) s.at_lead = atomicAdd(&lead.n_all, n);
        __syncthreads();
        const unsigned at = s.at_lead;
        for (unsigned i = tid; i < min(n, (unsigned) SM_LIST); i += SM_NT)
            if (at + i < SM_LIST) lead.list[at + i] = s.w[i];
        if (tid < C) cl.map_shared_rank(&s, tid)->all_n[rank] = n;
    };
    auto list_length = [&]() -> int { return (int) __reduce_add_sync(~0u, lane < C ? s.all_n[lane] : 0u); };

    // the row's whole mass, in full: every CTA's part summed, then the cluster's
    auto whole_mass = [&]() -> u64 {
        u64 sum = 0;
        for (int o = 0; o < p.seg; o += SM_TILE) {
            const uint4 q = *(const uint4 *) (mine + o);
            sum += weigh.raw4(q);   // the weight of -infinity is 0
        }
        sum -= (u64) (p.seg / 32) * Weigher::RAW;
        unsigned d0 = 0, d1;
        u64 t;
        scan2(s, d0, sum, d1, t);
        if (tid < C) cl.map_shared_rank(&s, tid)->all_mass[rank] = t;
        cl.sync();
        return sum8(lane < C ? s.all_mass[lane] : 0ull);
    };
    if (lists) {
        if (by_m) {          // what w >= m can reach, downwards by more than the roundings on the way
            const double lo = (double) xmax + (double) temp * log(m);
            floor = max(key_of((float) (lo - 1e-6 * (fabs(lo) + fabs((double) xmax) + (double) temp))), KEY_NONE + 1);
        }
        const float c2 = (float) weigh.c;
        float near = 0.0f, listed = 0.0f;   // the words' mass, and the listed words'
        for (int o = 0; o < p.seg; o += SM_TILE) {
            const uint4 q = *(const uint4 *) (mine + o);
            if (max(max(q.x, q.y), max(q.z, q.w)) >= floor)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t k = (&q.x)[e];
                    if (k >= floor) {
                        const unsigned at = atomicAdd(&s.n_list, 1u);
                        if (at < SM_LIST) s.w[at] = ((u64) k << 32) | (uint32_t) ~(uint32_t) (first + o + e);
                    }
                }
            if (by_p) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float y = __fmul_rn(__fadd_rn(value_of((&q.x)[i]), -xmax), c2);
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[i]) : "f"(y));
                }
                near = __fadd_rn(near, __fadd_rn(__fadd_rn(e[0], e[1]), __fadd_rn(e[2], e[3])));
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if ((&q.x)[i] >= floor) listed = __fadd_rn(listed, e[i]);
            }
        }
        if (by_p) {
            double t = (double) near, l = (double) listed;
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                t += __shfl_xor_sync(~0u, t, d);
                l += __shfl_xor_sync(~0u, l, d);
            }
            if (lane == 0) s.near[warp] = make_double2(t, l);
            __syncthreads();
            if (warp == 0) {
                double2 v = lane < SM_NW ? s.near[lane] : make_double2(0.0, 0.0);
#pragma unroll
                for (int d = 16; d; d >>= 1) {
                    v.x += __shfl_xor_sync(~0u, v.x, d);
                    v.y += __shfl_xor_sync(~0u, v.y, d);
                }
                if (lane < C) {   // to every CTA
                    SampleShared &o = *cl.map_shared_rank(&s, lane);
                    o.all_near[rank] = v.x;
                    o.all_listed[rank] = v.y;
                }
            }
        }
        push_list();
        cl.sync();
        const double nearW = by_p ? sum8(lane < C ? s.all_near[lane] : 0.0) * SM_ONE : 0.0;
        const double listedW = by_p ? sum8(lane < C ? s.all_listed[lane] : 0.0) * SM_ONE : 0.0;
        const int n = list_length();
        // certain already to go on below the list
        const bool below = by_p && listedW * (1.0 + SM_MASS_ERR) < pd * nearW * (1.0 - SM_MASS_ERR);
        if (!by_p && rank != 0 && n <= SM_LIST) return;   // nobody reads this CTA's shared memory any more
        if (n <= SM_LIST && !below) {
            if (!by_p) {
                weigh_list(n);
                if (n <= SM_SHORT) {
                    __syncthreads();
                    const Place at = place(n);
                    bool keep = at.in && (!use_k || at.rank < top_k);
                    if (use_p) {
                        if (at.in && at.rank == (use_k ? min(top_k, n) : n) - 1) s.total = at.after;
                        __syncthreads();
                        keep = keep && (at.rank == 0 || (double) at.before < pd * (double) s.total);
                    }
                    short_pick(n, keep);
                    return;
                }
                u64 last = 0;   // the last word kept
                if (use_k && n > top_k) {
                    by_score(n, 0, [](int) { return 1ull; }, [&](u64 b, u64 e) { return b < (u64) top_k && e >= (u64) top_k; });
                    last = s.found;
                }
                __syncthreads();
                if (use_p) {
                    unsigned d;
                    const double lim = pd * (double) list_mass(n, last, false, d);
                    by_score(n, 0, [&](int i) -> u64 { return s.list[i] >= last ? s.w[i] & ~PASS : 0; },
                             [&](u64 b, u64 e) { return (double) b < lim && (double) e >= lim; });
                    last = s.found;
                    __syncthreads();
                }
                pick(n, last);
                return;
            }
            // 0: the nucleus ends below the list, 1: it ends in it, 2: where it ends depends on the mass's error
            u64 last = 0, total = 0;
            Place at = {};
            const bool short_list = n <= SM_SHORT;
            auto to_mass = [&](double lim) {
                by_score(n, 0, whole_of, [&](u64 b, u64 e) { return (double) b < lim && (double) e >= lim; });
                last = s.found;
            };
            auto tell = [&](unsigned v) {   // the leading CTA's thread 0, to every CTA
                for (int r = 0; r < C; r++) cl.map_shared_rank(&s, r)->done = v;
            };
            auto before = [&](double lim) { return at.in && (at.rank == 0 || (double) at.before < lim); };
            if (rank == 0) {
                unsigned d;
                weigh_list(n);
                __syncthreads();
                const double lo = pd * nearW * (1.0 - SM_MASS_ERR), hi = pd * nearW * (1.0 + SM_MASS_ERR);
                bool sure;
                if (short_list) {
                    at = place(n);
                    if (at.in && at.rank == n - 1) s.total = at.after;
                    sure = !__syncthreads_or(before(lo) != before(hi));
                    total = s.total;
                    sure = sure && (double) total >= hi;
                } else {
                    total = list_mass(n, 0, false, d);
                    to_mass(lo);
                    sure = (double) s.found_after >= hi;
                }
                if (tid == 0) tell((double) total < lo ? 0 : sure ? 1 : 2);   // NaN: 2
            }
            cl.sync();
            const unsigned done = s.done;
            auto finish = [&](double lim) {
                if (short_list) short_pick(n, before(lim));
                else pick(n, last);
            };
            if (done == 1) {
                if (rank == 0) finish(pd * nearW);
                return;
            }
            if (done == 2) {
                const double lim = pd * (double) whole_mass();
                if (rank == 0) {
                    if (!short_list) to_mass(lim);
                    if (tid == 0) tell((double) total >= lim);
                }
                cl.sync();
                if (s.done) {
                    if (rank == 0) finish(lim);
                    return;
                }
            }
        }
        cl.sync();
    }

    // ---- the long way ----
    // for top-k the smallest key, and how many there are
    uint32_t mn = ~0u;
    unsigned nv = 0;
    if (use_k) {
        for (int o = 0; o < p.seg; o += SM_TILE) {
            const uint4 q = *(const uint4 *) (mine + o);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t k = (&q.x)[e];
                if (k > KEY_NONE) { mn = min(mn, k); nv++; }
            }
        }
        mn = __reduce_min_sync(~0u, mn);
        nv = __reduce_add_sync(~0u, nv);
        if (lane == 0) { atomicMin(&s.mn, mn); atomicAdd(&s.nvalid, nv); }
        cl.sync();
        mn = __reduce_min_sync(~0u, OF_CTAS(mn, ~0u));
        nv = __reduce_add_sync(~0u, OF_CTAS(nvalid, 0u));
    }
    // One search: the value T, and how many words c at T, at which the count reaches k (by_mass false) or the mass
    // reaches p of the total (true). Only keys above `over` count; `extra` more mass lies at `over` itself.
    float scale = 0.0f;
    auto bin0 = [&](uint32_t k) -> int {   // rounded by an addition: the conversion unit is slow. The largest, infinite too: 0
        const float y = fminf(fmaxf(__fmul_rn(__fadd_rn(xmax, -value_of(k)), scale), 0.0f), (float) (SM_BINS - 1));
        return (int) (__float_as_uint(__fadd_rn(y, 8388608.0f)) & (SM_BINS - 1));
    };
    // the list holds the last word kept: the one before which less than lim lies and with which lim is reached, of weights or
    // (by_mass false) of words. T and c of it to every CTA
    auto end_in_list = [&](int n, bool by_mass, u64 above, double lim, uint32_t &T, unsigned &c) {
        if (rank == 0) {
            weigh_list(n);
            __syncthreads();
            by_score(n, above, [&](int i) -> u64 { return by_mass ? s.w[i] & ~PASS : 1; },
                     [&](u64 b, u64 e) { return (double) b < lim && (double) e >= lim; });
            const u64 q = s.found;
            unsigned mine = 0;
            for (int i = tid; i < n; i += SM_NT) mine += s.list[i] >= q && s.list[i] >> 32 == q >> 32;
            u64 d0 = 0, d1;
            unsigned at;
            scan2(s, mine, d0, at, d1);
            if (tid < C) {   // to every CTA
                SampleShared &o = *cl.map_shared_rank(&s, tid);
                o.T = (uint32_t) (q >> 32);
                o.c = at;
            }
        }
        cl.sync();
        T = s.T;
        c = s.c;
    };
    auto search = [&](bool by_mass, uint32_t over, u64 extra, uint32_t &T, unsigned &c) {
        // the steps of level 0: down to the smallest score, or to where weights vanish; at most 64 (masked words of low values)
        const float range = fminf(by_mass ? temp * 31.2f : __fadd_rn(xmax, -value_of(mn)), 64.0f);
        scale = range > 0.0f ? fminf(__fdiv_rn((float) SM_BINS, range), 3e38f) : 0.0f;
        uint32_t klo = over + 1, khi = mx;        // keys still in question
        unsigned above = 0;                        // words, and mass, above khi
        u64 mass_above = 0;
        double lim = 0.0;
        int in_bin = -1;                           // level 0's bin the search is in
        for (int level = 0;; level++) {
            const u64 width = ((u64) khi - klo) / SM_BINS + 1;   // keys per bin from level 1 on
            auto bin_of = [&](uint32_t k) -> int {               // -1: not in question
                if (k < klo || k > khi) return -1;
                if (level == 0) return bin0(k);
                return bin0(k) == in_bin ? (int) ((khi - k) / (uint32_t) width) : -1;
            };
            for (int b = tid; b < SM_BINS; b += SM_NT) s.bins[0][b] = s.bins[1][b] = s.bins[2][b] = 0;
            if (tid == 0) { s.bin = -1; s.lo = ~0u; s.hi = 0; s.n_list = s.n_all = 0; }
            __syncthreads();
            for (int o = 0; o < p.seg; o += SM_TILE) {
                const uint4 q = *(const uint4 *) (mine + o);
                if (by_mass) {
                    double w[4];
                    weigh.four(q, w);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int b = bin_of((&q.x)[e]);
                        if (b < 0) continue;
                        const u64 wv = Weigher::whole(w[e]);
                        const unsigned d0 = (unsigned) wv & 32767, d1 = (unsigned) (wv >> 15) & 32767, d2 = (unsigned) (wv >> 30);
                        if (d0) atomicAdd(&s.bins[0][b], d0);
                        if (d1) atomicAdd(&s.bins[1][b], d1);
                        if (d2) atomicAdd(&s.bins[2][b], d2);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int b = bin_of((&q.x)[e]);
                        if (b >= 0) atomicAdd(&s.bins[0][b], 1u);
                    }
                }
            }
            cl.sync();
            // every CTA adds up all of them and finds the bin
            unsigned cn[2] = { 0, 0 };
            u64 ms[2] = { 0, 0 };
#pragma unroll
            for (int r = 0; r < SM_MAX_CLUSTER; r++)
                if (r < C) {
                    const SampleShared &o = *cl.map_shared_rank(&s, r);
                    const uint2 v = *(const uint2 *) &o.bins[0][2 * tid];
                    if (!by_mass) {
                        cn[0] += v.x;
                        cn[1] += v.y;
                    } else {
                        const uint2 v1 = *(const uint2 *) &o.bins[1][2 * tid], v2 = *(const uint2 *) &o.bins[2][2 * tid];
                        ms[0] += v.x + ((u64) v1.x << 15) + ((u64) v2.x << 30);
                        ms[1] += v.y + ((u64) v1.y << 15) + ((u64) v2.y << 30);
                    }
                }
            unsigned c0 = cn[0] + cn[1], tc;
            u64 m0 = ms[0] + ms[1], tm;
            scan2(s, c0, m0, tc, tm);
            if (by_mass && level == 0) lim = pd * (double) (tm + extra);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const unsigned ca = above + c0;
                const u64 ma = mass_above + m0;
                const bool here = by_mass ? (double) ma < lim && (double) (ma + ms[e]) >= lim && ms[e]
                                          : ca < (unsigned) top_k && ca + cn[e] >= (unsigned) top_k;
                if (here) {
                    s.bin = 2 * tid + e;
                    s.above = ca;
                    s.mass_above = ma;
                }
                c0 += cn[e];
                m0 += ms[e];
            }
            cl.sync();   // every CTA has read the histograms (whose memory the lists share) and knows the bin
            const int bin = s.bin;
            if (bin < 0) {   // by mass, the border lies among the words at `over`
                const u64 wt = weigh(over);
                T = over;
                c = wt ? (unsigned) fmax(1.0, ceil((lim - (double) (mass_above + tm)) / (double) wt)) : 0;
                cl.sync();   // read by all before it is written again (here and below)
                return;
            }
            above = s.above;
            mass_above = s.mass_above;
            if (level > 0 && width == 1) {   // one value
                T = khi - bin;
                if (by_mass) c = (unsigned) fmax(1.0, ceil((lim - (double) mass_above) / (double) weigh(T)));
                else c = top_k - above;
                cl.sync();
                return;
            }
            // the bin's words to a list
            for (int o = 0; o < p.seg; o += SM_TILE) {
                const uint4 q = *(const uint4 *) (mine + o);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t k = (&q.x)[e];
                    if (bin_of(k) != bin) continue;
                    const unsigned at = atomicAdd(&s.n_list, 1u);
                    if (at < SM_LIST) s.w[at] = ((u64) k << 32) | (uint32_t) ~(uint32_t) (first + o + e);
                }
            }
            push_list();
            cl.sync();
            const int nb = list_length();
            if (nb <= SM_LIST) {
                end_in_list(nb, by_mass, by_mass ? mass_above : above, by_mass ? lim : (double) top_k, T, c);
                return;
            }
            uint32_t l = ~0u, h = 0;   // too many: their range
            for (int o = 0; o < p.seg; o += SM_TILE) {
                const uint4 q = *(const uint4 *) (mine + o);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t k = (&q.x)[e];
                    if (bin_of(k) == bin) { l = min(l, k); h = max(h, k); }
                }
            }
            l = __reduce_min_sync(~0u, l);
            h = __reduce_max_sync(~0u, h);
            if (lane == 0) { atomicMin(&s.lo, l); atomicMax(&s.hi, h); }
            cl.sync();
            if (level == 0) in_bin = bin;
            klo = __reduce_min_sync(~0u, OF_CTAS(lo, ~0u));
            khi = __reduce_max_sync(~0u, OF_CTAS(hi, 0u));
            cl.sync();   // read by all before they are cleared
        }
    };

    uint32_t T = KEY_NONE;   // kept: keys above T, and the first c words at T (KEY_NONE: every valid word)
    unsigned c = 0;
    const bool cut = use_k && (unsigned) top_k < nv;
    if (cut) search(false, KEY_NONE, 0, T, c);
    if (use_p) {
        const uint32_t over = T;
        const u64 extra = cut ? c * weigh(T) : 0;
        uint32_t T2;
        unsigned c2;
        search(true, over, extra, T2, c2);
        c = T2 == T && cut ? min(c, c2) : c2;
        T = T2;
    }
    // the kept mass by id: per warp, then over the warps and the cluster
    u64 sum = 0;
    unsigned ties = 0, cnt = 0;
    const u64 wT = T > KEY_NONE ? weigh(T) : 0;
    const bool tie_in = T > KEY_NONE && (!use_m || T == mx || weigh.real(T) >= m);
    const bool ties_count = T > KEY_NONE;
    // the kept words above T among four: their weights (else 0), how many; and how many words at T
    auto take = [&](const uint4 &q, u64 (&w)[4], unsigned &kept, unsigned &at) {
        kept = at = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t k = (&q.x)[e];
            const double r = weigh.real(k);
            const bool in = k > T && (!use_m || k == mx || r >= m);
            w[e] = in ? Weigher::whole(r) : 0;
            kept += in;
            at += ties_count && k == T;
        }
    };
    if (!ties_count && !use_m) {   // no filter
        for (int o = 0; o < p.seg; o += SM_TILE) {
            const uint4 q = *(const uint4 *) (mine + o);
            sum += weigh.raw4(q);
            cnt += (q.x > KEY_NONE) + (q.y > KEY_NONE) + (q.z > KEY_NONE) + (q.w > KEY_NONE);
        }
        sum -= (u64) (p.seg / 32) * Weigher::RAW;
    } else {
        // the words above T are few: each warp queues them, and weighs 32 at once
        uint32_t *queue = s.queue[warp];
        int n = 0;
        __syncthreads();   // the lists in this memory are done with
        auto flush = [&](int have) {
            __syncwarp();
            const uint32_t k = lane < have ? queue[lane] : KEY_NONE;
            const double r = weigh.real(k);
            const bool in = k > KEY_NONE && (!use_m || k == mx || r >= m);
            sum += in ? Weigher::whole(r) : 0;
            cnt += in;
            const uint32_t rest = queue[32 + lane];
            __syncwarp();
            queue[lane] = rest;
            __syncwarp();
        };
        for (int o = 0; o < p.seg; o += SM_TILE) {
            const uint4 q = *(const uint4 *) (mine + o);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t k = (&q.x)[e];
                ties += ties_count && k == T;
                const unsigned in = __ballot_sync(~0u, k > T);
                if (!in) continue;
                if (k > T) queue[n + __popc(in & ((1u << lane) - 1))] = k;
                n += __popc(in);
                if (n >= 32) {
                    flush(32);
                    n -= 32;
                }
            }
        }
        flush(n);
    }
    ties = __reduce_add_sync(~0u, ties);
    cnt = __reduce_add_sync(~0u, cnt);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    // this warp's share in front of the CTA's later warps
    unsigned tb = lane == 0 ? ties : 0, tt;
    u64 sb = lane == 0 ? sum : 0, st;
    scan2(s, tb, sb, tt, st);
    tb = __shfl_sync(~0u, tb, 0);
    sb = __shfl_sync(~0u, sb, 0);
    if (tid == 0) { s.part_kept = 0; s.bin = -1; }
    __syncthreads();
    if (lane == 0) atomicAdd(&s.part_kept, cnt);
    __syncthreads();
    if (tid < C) {
        SampleShared &o = *cl.map_shared_rank(&s, tid);
        o.all_cnt[rank] = tt;
        o.all_sum[rank] = st;
        o.all_kept[rank] = s.part_kept;
    }
    cl.sync();
    const unsigned rt = lane < C ? s.all_cnt[lane] : 0u;
    const u64 rm = lane < C ? s.all_sum[lane] : 0ull;
    const unsigned all_ties = __reduce_add_sync(~0u, rt), all_cnt = __reduce_add_sync(~0u, lane < C ? s.all_kept[lane] : 0u);
    const u64 all = sum8(rm);
    tb += __reduce_add_sync(~0u, lane < rank ? rt : 0u);
    sb += sum8(lane < rank ? rm : 0ull);
    const unsigned ct = tie_in ? min(c, all_ties) : 0;
    const u64 kept_mass = all + ct * wT;
    const int kept = (int) (all_cnt + ct);
    const double target = (double) u * (double) kept_mass;
    auto mass_at = [&](u64 sum_, unsigned ties_) { return sum_ + min(ties_, ct) * wT; };
    // the warp whose share the target falls in is found; all warps of its CTA take its tiles, then one the tile's words
    if (lane == 0 && (double) mass_at(sb, tb) <= target && (double) mass_at(sb + sum, tb + ties) > target) {
        s.bin = warp;
        s.mass_above = sb;
        s.above = tb;
    }
    __syncthreads();
    const int cross = s.bin;
    if (cross >= 0) {
        uint32_t *seg = keys + cross * p.seg + 4 * lane;
        u64 b0 = s.mass_above;
        unsigned t0 = s.above;
        for (int o0 = 0; o0 < p.seg; o0 += SM_NW * SM_TILE) {   // rounds of a tile per warp
            const int o = o0 + warp * SM_TILE;
            const bool any = o < p.seg;
            u64 w[4] = { 0, 0, 0, 0 };
            unsigned n, lt = 0;
            uint4 q = make_uint4(0, 0, 0, 0);
            if (any) {
                q = *(const uint4 *) (seg + o);
                take(q, w, n, lt);
            }
            const u64 ls = (w[0] + w[1]) + (w[2] + w[3]);
            u64 b = ls, tm;
            unsigned bt = lt, tc;
            scan2(s, bt, b, tc, tm);
            b += b0;
            bt += t0;
            if (any && (double) mass_at(b, bt) <= target && (double) mass_at(b + ls, bt + lt) > target)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t k = (&q.x)[e];
                    const unsigned at = bt + (ties_count && k == T);
                    const u64 after = b + w[e];
                    if ((double) mass_at(b, bt) <= target && (double) mass_at(after, at) > target)
                        emit(base + cross * p.seg + 4 * lane + o + e, weigh.logprob(k, kept_mass), kept);
                    b = after;
                    bt = at;
                }
            b0 += tm;
            t0 += tc;
        }
    }
}

size_t sample_smem(int slice) { return (sizeof(SampleShared) + 15) / 16 * 16 + (size_t) slice * 4; }

}  // namespace

// the launch of checked arguments (the engine's sampling calls it too)
cudaError_t launch_sample(int device, const imi_cuda_sample_args &a, const void *const *rows, SessDev *const *states, cudaStream_t st) {
    const void *fn = a.type == IMI_F32   ? (const void *) k_sample<float>
                     : a.type == IMI_F16 ? (const void *) k_sample<__half>
                                          : (const void *) k_sample<__nv_bfloat16>;
    static SmemLimit lim;
    cudaError_t r = lim.raise(device, { (const void *) k_sample<float>, (const void *) k_sample<__half>, (const void *) k_sample<__nv_bfloat16> },
                              (int) sample_smem(SM_SLICE));
    const SampleSplit cut = sample_split(a.n, a.vocab);
    SampleArgs p = { a, cut.seg, cut.share, cut.rank, rows, states };
    void *args[] = { &p };
    if (r == cudaSuccess) r = launch_pdl(fn, dim3(a.n * cut.ctas), SM_NT, sample_smem(cut.seg * SM_NW), st, args, cut.ctas);
    return r;
}
}  // namespace imi

using namespace imi;

extern "C" imi_cuda_status imi_cuda_sample(int device, const imi_cuda_sample_args *a, void *stream) {
    if (!a || a->n < 0 || a->vocab < 1) return set_error(IMI_E_ARG, "sample: bad arguments");
    if (a->vocab > IMI_CUDA_SAMPLE_VOCAB)
        return set_error(IMI_E_ARG, "sample: at most " + std::to_string(IMI_CUDA_SAMPLE_VOCAB) + " words");
    if (a->type < IMI_F32 || a->type > IMI_BF16) return set_error(IMI_E_ARG, "sample: bad type");
    if (a->n == 0) return IMI_OK;
    if (a->n > 65535) return set_error(IMI_E_ARG, "sample: at most 65535 rows");
    if (!a->scores || !a->u || !a->ids) return set_error(IMI_E_ARG, "sample: null argument");
    if (a->stride < a->vocab && a->n > 1) return set_error(IMI_E_ARG, "sample: stride below vocab");
    if (!aligned(a->scores, a->type == IMI_F32 ? 4 : 2) || !aligned(a->u, 4) || !aligned(a->temperature, 4) || !aligned(a->top_k, 4) ||
        !aligned(a->top_p, 4) || !aligned(a->min_p, 4) || !aligned(a->ids, 4) || !aligned(a->logprob, 4) || !aligned(a->kept, 4))
        return set_error(IMI_E_ARG, "sample: a buffer is not aligned to its type");
    OnDevice on(device);
    if (!on.ok()) return set_error(IMI_E_NODEV, "no CUDA device " + std::to_string(device));
    if (!all_on_device({ a->scores, a->u, a->temperature, a->top_k, a->top_p, a->min_p, a->ids, a->logprob, a->kept }, device))
        return set_error(IMI_E_ARG, "sample: every buffer must be device memory of device " + std::to_string(device));
    const cudaError_t r = launch_sample(device, *a, nullptr, nullptr, (cudaStream_t) stream);
    if (r != cudaSuccess) return set_error(IMI_E_CUDA, std::string("sample: ") + cudaGetErrorString(r));
    return IMI_OK;
}
