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
//   The short way: while loading, every thread keeps its own words' maximum. The r-th largest of a CTA's thread maxima is
// a value that r of its words reach, so the smallest of these over the cluster, with r = ceil(k / CTAs), is one that k
// words reach; for top-p alone r is set for about 500 words, for min-p alone the value follows from the maximum. The few
// words above it are listed, and one CTA sorts them and applies the filters. Top-p's total mass is summed meanwhile.
//   The long way, where the list would be too long or ends inside the nucleus: a histogram over 1,024 steps of score
// (counts, masses), whose crossing bin is sorted by one CTA; a bin too full for that (masked words, all scores alike) is
// cut again, by keys. Then every CTA sums its kept words by id.
#include "common.cuh"
#include "serve.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace imi {
namespace {

constexpr int SM_NT = 512, SM_NW = SM_NT / 32;
constexpr int SM_BINS = 2 * SM_NT;       // two bins per thread in the scans
constexpr int SM_LIST = 1024;            // words one CTA sorts at most
constexpr int SM_AIM = 512;              // words listed for top-p alone, about
constexpr int SM_TILE = 128;             // words of a warp's load: four per lane
constexpr int SM_MAX_CLUSTER = 8;
constexpr int SM_SLICE = 32768;          // words a CTA holds at most
constexpr double SM_ONE = 17592186044416.0;   // 2^44
constexpr double SM_FAR = 31.2;          // exp(-31.2) < 2^-45: such a word's weight rounds to 0
constexpr int SM_TAB = 64;               // steps of the exponential's table
static_assert((long long) SM_SLICE * SM_MAX_CLUSTER >= IMI_CUDA_SAMPLE_VOCAB, "a row fits a cluster");
static_assert((long long) IMI_CUDA_SAMPLE_VOCAB <= 1 << 18, "the weights' sum fits 62 bits");

typedef unsigned long long u64;

struct SampleArgs {
    imi_cuda_sample_args a;
    int seg, slice;   // words per warp (a multiple of SM_TILE) and per CTA (SM_NW * seg)
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

// the same as a 64-bit number, by integer operations: the conversion unit takes about eight times as long for one. Numbers
// below 2^-126 become 0; infinity becomes a number (the callers look at the key).
__device__ __forceinline__ double wide_of(uint32_t k) {
    const uint32_t b = k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu), r = b & 0x7FFFFFFFu;
    const uint32_t hi = r >= 0x00800000u ? (b & 0x80000000u) | ((r >> 3) + 0x38000000u) : 0u;
    return __hiloint2double((int) hi, (int) (b << 29));
}

struct SampleShared {
    union {
        struct {
            unsigned cnt[SM_BINS], mass[SM_BINS][2];   // this CTA's histogram; mass: low and high words
        };
        struct {
            u64 list[SM_LIST], w[SM_LIST];   // (key, ~id) listed; weights in the list's order
        };
    };
    double tab[SM_TAB];               // 2^(i / 64)
    unsigned wc[SM_NW];               // scans over the CTA
    u64 wm[SM_NW];
    // what the cluster reads of this CTA
    u64 part_mass;
    unsigned part_cnt, part_kept, mx, mn, nvalid, floor, idmin, n_list, lo, hi;
    u64 mass_above;
    int bin;                          // found in a scan: the crossing bin, and what lies above it
    unsigned above, in_bin;
    unsigned T, c, done;              // the leading CTA's findings
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

// A word's weight, as a number and as an integer of 2^-44. exp by table (Tang, ACM TOMS 15, 1989): with n the nearest
// integer to z 64 / ln 2, exp(-z) = 2^(-n / 64) exp(r), r = n ln2 / 64 - z, |r| <= ln2 / 128, exp(r) to r^5 / 120 (the next
// term is below 2^-54). n reaches 2,881 here, so the rounding of ln2 / 64 costs 2^-48 of a weight that is itself 2^-45 then.
struct Weigher {
    double xmax;
    uint32_t kmax;
    double inv;   // 1 / temperature
    const double *tab;
    __device__ __forceinline__ double real(uint32_t k) const {   // no branches: several words are in flight at once
        const double z = (xmax - wide_of(k)) * inv;
        constexpr double MAGIC = 6755399441055744.0;   // 1.5 * 2^52: adding it leaves the nearest integer in the low bits
        const double b = __fma_rn(z, -64.0 * 1.4426950408889634074, MAGIC);
        const int n = __double2loint(b);               // <= 0
        const double r = __fma_rn(__dadd_rn(b, -MAGIC), -0.69314718055994530942 / 64.0, -z);
        double e = __fma_rn(r, 1.0 / 120.0, 1.0 / 24.0);
        e = __fma_rn(r, e, 1.0 / 6.0);
        e = __fma_rn(r, e, 0.5);
        e = __fma_rn(r, e, 1.0);
        e = __fma_rn(r, e, 1.0);
        e = __dmul_rn(e, tab[n & (SM_TAB - 1)]);
        e = __hiloint2double(__double2hiint(e) + (n >> 6) * (1 << 20), __double2loint(e));
        return k == kmax ? 1.0 : z < SM_FAR && k > KEY_NONE ? e : 0.0;
    }
    static __device__ __forceinline__ u64 whole(double w) {
        // w * 2^44 <= 2^44: added to 2^52 its integer part, rounded to nearest, is the low mantissa
        return (u64) __double_as_longlong(__fma_rn(w, SM_ONE, 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ u64 operator()(uint32_t k) const { return whole(real(k)); }
    __device__ __forceinline__ float logprob(uint32_t k, u64 total) const {
        const double z = k == kmax ? 0.0 : (xmax - (double) value_of(k)) * inv;
        return (float) (-z - log((double) total / SM_ONE));
    }
};

// v[0..n) sorted descending (all different, n at most SM_LIST, room up to the next power of two)
__device__ __forceinline__ void sort_desc(u64 *v, int n) {
    const int tid = threadIdx.x;
    if (n <= 256) {   // each value's place counted: a pass over n values, against 36 exchanges with a barrier each
        u64 x = 0;
        int place = 0;
        if (tid < n) {
            x = v[tid];
#pragma unroll 8
            for (int j = 0; j < n; j++) place += v[j] > x;
        }
        __syncthreads();
        if (tid < n) v[place] = x;
        __syncthreads();
        return;
    }
    int n2 = 512;
    while (n2 < n) n2 <<= 1;
    for (int i = n + tid; i < n2; i += SM_NT) v[i] = 0;
    __syncthreads();
    for (int k = 2; k <= n2; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = tid; i < n2 / 2; i += SM_NT) {
                const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                const u64 x = v[lo], y = v[hi];
                if ((x < y) == ((lo & k) == 0)) { v[lo] = y; v[hi] = x; }
            }
            __syncthreads();
        }
}

template <typename S>
__device__ __forceinline__ float score_at(const S *x, int i) {
    if constexpr (sizeof(S) == 4) return x[i];
    else if constexpr (std::is_same<S, __half>::value) return __half2float(x[i]);
    else return __bfloat162float(x[i]);
}

template <typename S>
__device__ __forceinline__ void load4(const S *x, float (&f)[4]) {
    if constexpr (sizeof(S) == 4) {
        const float4 v = __ldg((const float4 *) x);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    } else {
        const uint2 v = __ldg((const uint2 *) x);
#pragma unroll
        for (int e = 0; e < 4; e++) f[e] = score_at((const S *) &v, e);
    }
}

// a value of every CTA of the cluster: lane r holds CTA r's (other lanes `none`), read at once
#define OF_CTAS(field, none) (lane < C ? cl.map_shared_rank(&s, lane)->field : (none))
__device__ __forceinline__ u64 sum8(u64 v) {   // over the first 8 lanes, to all
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
    const int base = rank * p.slice;                       // this CTA's first word
    if (tid == 0) { s.mx = 0; s.mn = ~0u; s.nvalid = 0; s.idmin = ~0u; s.n_list = 0; s.floor = KEY_NONE + 1; }
    if (tid < SM_TAB) s.tab[tid] = exp2((double) tid / SM_TAB);
    __syncthreads();
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
    const S *x = (const S *) a.scores + row * a.stride;
    const bool vec = ((uintptr_t) (x + base) & (4 * sizeof(S) - 1)) == 0;
    uint32_t mx = 0;
    uint32_t *mine = keys + warp * p.seg + 4 * lane;        // the words of a lane, tile by tile
    const int first = base + warp * p.seg + 4 * lane;
    auto put = [&](int o, const float (&f)[4]) {
        uint4 k = make_uint4(key_of(f[0]), key_of(f[1]), key_of(f[2]), key_of(f[3]));
        mx = max(max(mx, max(k.x, k.y)), max(k.z, k.w));
        *(uint4 *) (mine + o) = k;
    };
    const int inside = a.vocab - (base + warp * p.seg);     // words of the row in this warp's part
    const int whole = vec ? max(0, min(p.seg, inside / SM_TILE * SM_TILE)) : 0;
    int o = 0;
    for (; o + 4 * SM_TILE <= whole; o += 4 * SM_TILE) {    // four tiles' loads in flight
        float f[4][4];
#pragma unroll
        for (int t = 0; t < 4; t++) load4(x + first + o + t * SM_TILE, f[t]);
#pragma unroll
        for (int t = 0; t < 4; t++) put(o + t * SM_TILE, f[t]);
    }
    for (; o < p.seg; o += SM_TILE) {
        float f[4];
        if (o < whole) load4(x + first + o, f);
        else
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = first + o + e < a.vocab ? score_at(x, first + o + e) : -INFINITY;
        put(o, f);
    }
    // the r-th largest of the threads' maxima, to 20 bits downwards
    const bool by_k = use_k && top_k <= SM_LIST, by_p = !use_k && use_p, by_m = !use_k && !use_p && use_m;
    const int r_th = by_k ? (top_k + C - 1) / C : by_p ? SM_AIM / C : 0;
    const bool lists = !greedy && r_th <= SM_NT && (by_k || by_p || by_m);
    uint32_t floor = 0;
    if (lists && r_th)
        for (int b = 31; b >= 12; b--)
            if (__syncthreads_count(mx >= (floor | 1u << b)) >= r_th) floor |= 1u << b;
    const uint32_t wmax = __reduce_max_sync(~0u, mx);
    if (lane == 0) atomicMax(&s.mx, wmax);
    if (tid == 0) s.floor = max(floor, KEY_NONE + 1);
    cl.sync();
    mx = __reduce_max_sync(~0u, OF_CTAS(mx, 0u));
    floor = __reduce_min_sync(~0u, OF_CTAS(floor, ~0u));
    auto emit = [&](int id, float lp, int kept) {
        a.ids[row] = id;
        if (a.logprob) a.logprob[row] = lp;
        if (a.kept) a.kept[row] = kept;
    };
    if (mx <= KEY_NONE) {
        if (rank == 0 && tid == 0) emit(-1, -INFINITY, 0);
        cl.sync();   // no CTA leaves while another may read its shared memory
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
        if (lane == 0) atomicMin(&s.idmin, id);
        cl.sync();
        id = __reduce_min_sync(~0u, OF_CTAS(idmin, ~0u));
        if (rank == 0 && tid == 0) emit((int) id, 0.0f, 1);
        cl.sync();
        return;
    }
    const Weigher weigh = { (double) xmax, mx, 1.0 / (double) temp, s.tab };

    // The list of n words, which reaches down to some value, ends the row if all that can be kept is in it: the filters, and
    // the pick by id. of_all: the mass that top-p's share is of where top-k does not cut the list. False: the nucleus goes on
    // below the list.
    auto finish_list = [&](int n, u64 of_all) -> bool {
        sort_desc(s.list, n);
        if (use_k) n = min(n, top_k);
        // two words per thread: weights, their sums, and how many pass
        u64 wv[2], sum = 0;
        unsigned pass = 0;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int j = 2 * tid + e;
            const double w = j < n ? weigh.real((uint32_t) (s.list[j] >> 32)) : 0.0;
            wv[e] = j < n ? Weigher::whole(w) : 0;
            if (j < n) s.w[j] = wv[e];
            if (j < n && (!use_m || j == 0 || w >= m)) pass++;
            sum += wv[e];
        }
        unsigned ex = pass, tp;
        u64 before = sum, total;
        scan2(s, ex, before, tp, total);
        int K = (int) tp;
        if (use_p) {
            const double lim = pd * (double) (use_k ? total : of_all);
            if (!use_k && (double) total < lim) return false;
            unsigned keep = 0, all;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int j = 2 * tid + e;
                if (j < n && (j == 0 || (double) before < lim)) keep++;
                before += wv[e];
            }
            u64 d0 = 0, d1;
            scan2(s, keep, d0, all, d1);
            K = min(K, (int) all);
        }
        __syncthreads();
        if (K <= 128) {   // each word's running sum by id counted directly
            u64 b = 0, t = 0, q = 0, w = 0;
            if (tid < K) {
                q = s.list[tid];
                w = s.w[tid];
#pragma unroll 4
                for (int j = 0; j < K; j++) {
                    const u64 wj = s.w[j];
                    t += wj;
                    if ((unsigned) s.list[j] > (unsigned) q) b += wj;   // ~id larger: id smaller
                }
                const double target = (double) u * (double) t;
                if ((double) b <= target && (double) (b + w) > target)
                    emit((int) ~(unsigned) q, weigh.logprob((uint32_t) (q >> 32), t), K);
            }
            return true;
        }
        // by id: (~id, place in the order of scores) sorted descending
        for (int j = tid; j < K; j += SM_NT) s.list[j] = s.list[j] << 32 | (unsigned) j;
        __syncthreads();
        sort_desc(s.list, K);
        sum = 0;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int j = 2 * tid + e;
            wv[e] = j < K ? s.w[(unsigned) s.list[j]] : 0;
            sum += wv[e];
        }
        unsigned d0 = 0, d1;
        before = sum;
        scan2(s, d0, before, d1, total);
        const double target = (double) u * (double) total;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int j = 2 * tid + e;
            const u64 after = before + wv[e];
            if (j < K && (double) before <= target && (double) after > target) {
                const int id = (int) ~(unsigned) (s.list[j] >> 32);
                emit(id, weigh.logprob(key_of(score_at(x, id)), total), K);
            }
            before = after;
        }
        return true;
    };

    // the CTAs' lists: how many words together, and all of them to the leading CTA's
    auto collect_count = [&]() -> unsigned { return __reduce_add_sync(~0u, OF_CTAS(n_list, 0u)); };
    auto collect = [&]() {
        const unsigned c = OF_CTAS(n_list, 0u);
        unsigned before = c;
#pragma unroll
        for (int d = 1; d < SM_MAX_CLUSTER; d <<= 1) {
            const unsigned y = __shfl_up_sync(~0u, before, d);
            if (lane >= d) before += y;
        }
        before -= c;
        const int r = warp % SM_MAX_CLUSTER;   // two warps per CTA of the cluster
        const unsigned at = __shfl_sync(~0u, before, r), n = __shfl_sync(~0u, c, r);
        if (r > 0 && r < C) {
            const SampleShared &o = *cl.map_shared_rank(&s, r);
            for (unsigned i = (warp / SM_MAX_CLUSTER) * 32 + lane; i < n; i += SM_NT / SM_MAX_CLUSTER) s.list[at + i] = o.list[i];
        }
        __syncthreads();
    };

    u64 W0 = 0;              // the row's whole mass, where the short way has summed it
    if (lists) {
        if (by_m) {          // what w >= m can reach, downwards by more than the roundings on the way
            const double lo = (double) xmax + (double) temp * log(m);
            floor = max(key_of((float) (lo - 1e-6 * (fabs(lo) + fabs((double) xmax) + (double) temp))), KEY_NONE + 1);
        }
        u64 sum = 0;
        for (int o = 0; o < p.seg; o += SM_TILE) {
            const uint4 q = *(const uint4 *) (mine + o);
            if (max(max(q.x, q.y), max(q.z, q.w)) >= floor)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t k = (&q.x)[e];
                    if (k >= floor) {
                        const unsigned at = atomicAdd(&s.n_list, 1u);
                        if (at < SM_LIST) s.list[at] = ((u64) k << 32) | (uint32_t) ~(uint32_t) (first + o + e);
                    }
                }
            if (by_p) {   // the weight of -infinity is 0
                const u64 w0 = weigh(q.x), w1 = weigh(q.y), w2 = weigh(q.z), w3 = weigh(q.w);
                sum += (w0 + w1) + (w2 + w3);
            }
        }
        if (by_p) {
            unsigned d0 = 0, d1;
            u64 t;
            scan2(s, d0, sum, d1, t);
            if (tid == 0) s.part_mass = t;
        }
        cl.sync();
        if (by_p) W0 = sum8(OF_CTAS(part_mass, 0ull));
        const unsigned n = collect_count();
        if (n <= SM_LIST) {
            if (rank == 0) collect();
            if (!by_p) {
                cl.sync();   // the lists have been read
                if (rank == 0) finish_list((int) n, 0);
                return;
            }
            if (rank == 0) {
                const bool ok = finish_list((int) n, W0);
                if (tid == 0) s.done = ok;
            }
            cl.sync();
            if (cl.map_shared_rank(&s, 0)->done) {
                cl.sync();
                return;
            }
        }
        cl.sync();
    }

    // ---- the long way ----
    // the smallest key, and how many there are
    if (use_k || use_p) {
        uint32_t mn = ~0u;
        unsigned nv = 0;
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
    }
    const uint32_t mn = __reduce_min_sync(~0u, OF_CTAS(mn, ~0u));
    const unsigned nv = __reduce_add_sync(~0u, OF_CTAS(nvalid, 0u));
    // One search: the value T, and how many words c at T, at which the count reaches k (by_mass false) or the mass
    // reaches p of the total (true). Only keys above `over` count; `extra` more mass lies at `over` itself.
    const float range = fminf(__fadd_rn(xmax, -value_of(mn)), 64.0f);
    const float scale = range > 0.0f ? __fdiv_rn((float) SM_BINS, range) : 0.0f;
    auto search = [&](bool by_mass, uint32_t over, u64 extra, uint32_t &T, unsigned &c) {
        uint32_t klo = over + 1, khi = mx;        // keys still in question
        unsigned above = 0;                        // words, and mass, above khi
        u64 mass_above = 0;
        double lim = 0.0;
        int in_bin = -1;                           // level 0's bin the search is in
        for (int level = 0;; level++) {
            auto bin0 = [&](uint32_t k) -> int {
                if (k == mx) return 0;
                return min(SM_BINS - 1, __float2int_rz(__fmul_rn(__fadd_rn(xmax, -value_of(k)), scale)));
            };
            const u64 width = ((u64) khi - klo) / SM_BINS + 1;   // keys per bin from level 1 on
            auto bin_of = [&](uint32_t k) -> int {               // -1: not in question
                if (k < klo || k > khi) return -1;
                if (level == 0) return bin0(k);
                return bin0(k) == in_bin ? (int) ((khi - k) / (uint32_t) width) : -1;
            };
            for (int b = tid; b < SM_BINS; b += SM_NT) s.cnt[b] = s.mass[b][0] = s.mass[b][1] = 0;
            if (tid == 0) { s.bin = -1; s.lo = ~0u; s.hi = 0; s.n_list = 0; }
            __syncthreads();
            for (int o = 0; o < p.seg; o += SM_TILE) {
                const uint4 q = *(const uint4 *) (mine + o);
                u64 wv[4];
                if (by_mass)
#pragma unroll
                    for (int e = 0; e < 4; e++) wv[e] = weigh((&q.x)[e]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int b = bin_of((&q.x)[e]);
                    if (b < 0) continue;
                    atomicAdd(&s.cnt[b], 1u);
                    if (by_mass) {   // 64-bit addition by halves: the carry is what the low half's old value shows
                        const u64 w = wv[e];
                        const unsigned wl = (unsigned) w, old = atomicAdd(&s.mass[b][0], wl);
                        const unsigned wh = (unsigned) (w >> 32) + (old + wl < old);
                        if (wh) atomicAdd(&s.mass[b][1], wh);
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
                    const uint2 v = *(const uint2 *) &o.cnt[2 * tid];
                    cn[0] += v.x;
                    cn[1] += v.y;
                    if (by_mass) {
                        const uint4 w = *(const uint4 *) &o.mass[2 * tid][0];
                        ms[0] += (u64) w.y << 32 | w.x;
                        ms[1] += (u64) w.w << 32 | w.z;
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
                    s.in_bin = cn[e];
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
            const unsigned nb = s.in_bin;
            if (level > 0 && width == 1) {   // one value
                T = khi - bin;
                if (by_mass) c = (unsigned) fmax(1.0, ceil((lim - (double) mass_above) / (double) weigh(T)));
                else c = top_k - above;
                c = min(c, nb);
                cl.sync();
                return;
            }
            // the bin's words to a list; their range where they are too many
            const bool fits = nb <= SM_LIST;
            for (int o = 0; o < p.seg; o += SM_TILE) {
                const uint4 q = *(const uint4 *) (mine + o);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t k = (&q.x)[e];
                    if (bin_of(k) != bin) continue;
                    if (fits) {
                        const unsigned at = atomicAdd(&s.n_list, 1u);
                        if (at < SM_LIST) s.list[at] = ((u64) k << 32) | (uint32_t) ~(uint32_t) (first + o + e);
                    } else {
                        atomicMin(&s.lo, k);
                        atomicMax(&s.hi, k);
                    }
                }
            }
            cl.sync();
            if (fits) {
                if (rank == 0) {
                    const unsigned n = collect_count();
                    collect();
                    sort_desc(s.list, (int) n);
                    u64 wv[2] = { 0, 0 };
                    unsigned dc = 0, dt;
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if (by_mass && 2 * tid + e < (int) n) wv[e] = weigh((uint32_t) (s.list[2 * tid + e] >> 32));
                    u64 bm = wv[0] + wv[1], bt;
                    scan2(s, dc, bm, dt, bt);
                    bm += mass_above;
#pragma unroll
                    for (int e = 0; e < 2; e++) {   // the last word kept: T is its value, c its place among those of T
                        const int j = 2 * tid + e;
                        const bool lastk = by_mass ? j < (int) n && (double) bm < lim && ((double) (bm + wv[e]) >= lim || j + 1 == (int) n)
                                                   : j == top_k - 1 - (int) above;
                        if (lastk) {
                            const uint32_t key = (uint32_t) (s.list[j] >> 32);
                            int f = j;
                            while (f > 0 && (uint32_t) (s.list[f - 1] >> 32) == key) f--;
                            s.T = key;
                            s.c = j - f + 1;
                        }
                        bm += wv[e];
                    }
                }
                cl.sync();
                const SampleShared &lead = *cl.map_shared_rank(&s, 0);
                T = lead.T;
                c = lead.c;
                cl.sync();
                return;
            }
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
        w[0] = w[1] = w[2] = w[3] = 0;
        kept = at = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) at += ties_count && (&q.x)[e] == T;
        if (max(max(q.x, q.y), max(q.z, q.w)) <= T) return;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t k = (&q.x)[e];
            const double r = weigh.real(k);
            const bool in = k > T && (!use_m || k == mx || r >= m);
            w[e] = in ? Weigher::whole(r) : 0;
            kept += in;
        }
    };
    for (int o = 0; o < p.seg; o += SM_TILE) {
        u64 w[4];
        unsigned kept, at;
        take(*(const uint4 *) (mine + o), w, kept, at);
        sum += (w[0] + w[1]) + (w[2] + w[3]);
        cnt += kept;
        ties += at;
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
    if (tid == 0) { s.part_cnt = tt; s.part_mass = st; s.part_kept = 0; s.bin = -1; }
    __syncthreads();
    if (lane == 0) atomicAdd(&s.part_kept, cnt);
    cl.sync();
    const unsigned rt = OF_CTAS(part_cnt, 0u);
    const u64 rm = OF_CTAS(part_mass, 0ull);
    const unsigned all_ties = __reduce_add_sync(~0u, rt), all_cnt = __reduce_add_sync(~0u, OF_CTAS(part_kept, 0u));
    const u64 all = sum8(rm);
    tb += __reduce_add_sync(~0u, lane < rank ? rt : 0u);
    sb += sum8(lane < rank ? rm : 0ull);
    const unsigned ct = tie_in ? min(c, all_ties) : 0;
    const u64 W = all + ct * wT;
    const int kept = (int) (all_cnt + ct);
    const double target = (double) u * (double) W;
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
                        emit(base + cross * p.seg + 4 * lane + o + e, weigh.logprob(k, W), kept);
                    b = after;
                    bt = at;
                }
            b0 += tm;
            t0 += tc;
        }
    }
    cl.sync();
}

size_t sample_smem(int slice) { return (sizeof(SampleShared) + 15) / 16 * 16 + (size_t) slice * 4; }

}  // namespace
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
    const void *fn = a->type == IMI_F32   ? (const void *) k_sample<float>
                     : a->type == IMI_F16 ? (const void *) k_sample<__half>
                                          : (const void *) k_sample<__nv_bfloat16>;
    static SmemLimit lim;
    cudaError_t r = lim.raise(device, { (const void *) k_sample<float>, (const void *) k_sample<__half>, (const void *) k_sample<__nv_bfloat16> },
                              (int) sample_smem(SM_SLICE));
    // CTAs per row: as many as hold the row, more while the rows leave SMs idle and a CTA keeps a tile per warp
    int C = 1;
    while (C < SM_MAX_CLUSTER && ((a->vocab + C - 1) / C > SM_SLICE || (a->n * C < 148 && a->vocab > C * SM_NW * SM_TILE))) C *= 2;
    SampleArgs p = { *a, 0, 0 };
    p.seg = ((a->vocab + C * SM_NW - 1) / (C * SM_NW) + SM_TILE - 1) / SM_TILE * SM_TILE;
    p.slice = p.seg * SM_NW;
    void *args[] = { &p };
    if (r == cudaSuccess) r = launch_pdl(fn, dim3(a->n * C), SM_NT, sample_smem(p.slice), (cudaStream_t) stream, args, C);
    if (r != cudaSuccess) return set_error(IMI_E_CUDA, std::string("sample: ") + cudaGetErrorString(r));
    return IMI_OK;
}
