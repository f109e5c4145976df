// Serving operators over pages: block tables and slot maps made from the requests' lengths (imi_cuda_page_map) and K and V
// rows written to the slots (imi_cuda_page_write).
#include "common.cuh"
#include "serve.h"

#include <cuda_bf16.h>

#include <algorithm>

namespace imi {
namespace {

constexpr int MAP_ROWS = 4096, MAP_THREADS = 512;

struct MapArgs {
    imi_cuda_page_map_args a;
    int shift;   // log2(page)
};

// the largest i of 0..n-1 with first[i] <= j (first non-decreasing, first[0] = 0)
__device__ __forceinline__ int row_of(const int *first, int n, int j) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= j) lo = mid;
        else hi = mid;
    }
    return lo;
}

// With have = ceil(held / page), need = ceil((held + add) / page) - have and first the exclusive sum of need, the new
// page c >= have of request i is free[n_free - 1 - (first_i + c - have_i)]; token t of the step belongs to the request
// with start_i <= t < start_{i+1} and sits at position p = held_i + t - start_i.
// Bound by launch latency and one round trip for the lengths at decode sizes, by the 8 bytes written per new row at
// the largest. Every CTA scans all lengths itself (8 n bytes from L2, at most 32 KB): no CTA waits for another, and
// the table entries, slots and positions are then shared out evenly. What may alias an input (length, n_free_out) is
// written by the CTA that is the last to have read its inputs; the count of those that have is asked for before the tables
// and slots are written, and its answer used after that. A CTA has read all of them by the scan's barrier; fences in front of
// its count and behind the last one's order those reads before the writes.
// Measured, one call behind the other: 64 decode steps 5.0 us, 384 prompts of 1,000,000 tokens at most (8 MB written) 10.2 to 11.4.
__global__ void __launch_bounds__(MAP_THREADS) k_page_map(const __grid_constant__ MapArgs m) {
    extern __shared__ int sh[];
    const imi_cuda_page_map_args &a = m.a;
    const int n = a.n, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int *held = sh, *start = sh + n, *first = start + n + 1;
    __shared__ long long ws[2][MAP_THREADS / 32];
    __shared__ int werr[MAP_THREADS / 32], last, free_now;
    pdl_wait();
    pdl_trigger();
    if (tid == 0) free_now = *a.n_free;
    // each thread: `per` consecutive requests, then a scan of the threads' sums
    const int per = (n + MAP_THREADS - 1) / MAP_THREADS, i0 = min(n, tid * per), i1 = min(n, i0 + per);
    long long sa = 0, sn = 0;
    int err = 0;
    for (int i = i0; i < i1; i++) {
        const int h = a.held[i], ad = h < 0 ? 0 : a.add[i];
        held[i] = h;
        if (ad < 0) err = max(err, (int) IMI_DEV_LENGTH);
        const long long tot = h < 0 ? 0 : (long long) h + max(ad, 0);
        if (tot > (long long) a.width << m.shift) err = max(err, (int) IMI_DEV_TABLE);
        const long long have = h < 0 ? 0 : ((long long) h + a.page - 1) >> m.shift;
        first[i] = (int) (((tot + a.page - 1) >> m.shift) - have);   // need, summed below (h < 0: 0)
        start[i] = max(ad, 0);
        sa += start[i];
        sn += first[i];
    }
    long long xa = sa, xn = sn;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long ya = __shfl_up_sync(~0u, xa, o), yn = __shfl_up_sync(~0u, xn, o);
        if (lane >= o) { xa += ya; xn += yn; }
    }
    err = __reduce_max_sync(~0u, err);
    if (lane == 31) { ws[0][warp] = xa; ws[1][warp] = xn; werr[warp] = err; }
    __syncthreads();
    const int n_free = free_now;
    long long ba = 0, bn = 0, ta = 0, tn = 0;
    err = 0;
#pragma unroll
    for (int w = 0; w < MAP_THREADS / 32; w++) {
        if (w < warp) { ba += ws[0][w]; bn += ws[1][w]; }
        ta += ws[0][w];
        tn += ws[1][w];
        err = max(err, werr[w]);
    }
    if (ta > a.cap) err = max(err, (int) IMI_DEV_CAP);
    if (n_free < 0 || n_free > a.free_cap || tn > n_free) err = max(err, (int) IMI_DEV_POOL);
    long long ea = ba + xa - sa, en = bn + xn - sn;   // exclusive sums in front of this thread
    const bool ok = err == 0;
    for (int i = i0; i < i1; i++) {
        const int ad = start[i], nd = first[i];
        start[i] = ok ? (int) ea : 0;
        first[i] = ok ? (int) en : 0;
        ea += ad;
        en += nd;
    }
    const int rows = ok ? (int) ta : 0, pages = ok ? (int) tn : 0;
    int read = 0;   // thread 0: CTAs that had read their inputs before this one (whose threads all have, since the scan)
    if (tid == 0) {
        start[n] = rows;
        if (gridDim.x > 1) {
            __threadfence();
            read = atomicAdd(a.status + 1, 1);
        }
    }
    __syncthreads();
    bool bad = false;
    // the new table entries
    for (int j = blockIdx.x * MAP_THREADS + tid; j < pages; j += gridDim.x * MAP_THREADS) {
        const int i = row_of(first, n, j), id = a.free_pages[n_free - 1 - j];
        const int c = ((held[i] + a.page - 1) >> m.shift) + j - first[i];
        a.table[i * a.table_stride + c] = id;
        bad |= (unsigned) id >= (unsigned) a.n_pages;
    }
    // slots and positions, four rows per thread (one search, then forward from request to request)
    for (long long t0 = 4LL * (blockIdx.x * MAP_THREADS + tid); t0 < a.cap; t0 += 4LL * gridDim.x * MAP_THREADS) {
        int i = t0 < rows ? row_of(start, n, (int) t0) : 0, sl[4], ps[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const long long t = t0 + k;
            sl[k] = ps[k] = -1;
            if (t >= rows) continue;
            while (start[i + 1] <= t) i++;   // ends: start[n] = rows > t
            const int p = held[i] + (int) t - start[i], c = p >> m.shift, have = (held[i] + a.page - 1) >> m.shift;
            const int id = c < have ? a.table[i * a.table_stride + c] : a.free_pages[n_free - 1 - (first[i] + c - have)];
            if ((unsigned) id < (unsigned) a.n_pages) sl[k] = (id << m.shift) + (p & (a.page - 1));
            else bad = true;
            ps[k] = a.pos0 + p;
        }
        if (t0 + 4 <= a.cap && ((((uintptr_t) a.slots) | ((uintptr_t) a.pos)) & 15) == 0) {
            *(int4 *) (a.slots + t0) = make_int4(sl[0], sl[1], sl[2], sl[3]);
            *(int4 *) (a.pos + t0) = make_int4(ps[0], ps[1], ps[2], ps[3]);
        } else {
            for (int k = 0; k < 4 && t0 + k < a.cap; k++) { a.slots[t0 + k] = sl[k]; a.pos[t0 + k] = ps[k]; }
        }
    }
    if (bad) atomicMax(a.status, IMI_DEV_PAGE);
    if (gridDim.x > 1) {
        if (tid == 0) {
            last = read == (int) gridDim.x - 1;
            if (last) __threadfence();
        }
        __syncthreads();
        if (!last) return;
    }
    for (int i = tid; i < n; i += MAP_THREADS) {
        a.start[i] = start[i];
        a.length[i] = ok && held[i] >= 0 ? held[i] + start[i + 1] - start[i] : held[i] < 0 ? -1 : held[i];
    }
    if (tid == 0) {
        a.start[n] = rows;
        *a.n_free_out = n_free - pages;
        if (err) atomicMax(a.status, err);
        if (gridDim.x > 1) a.status[1] = 0;
    }
}

// ---- page_write ----
struct WriteArgs {
    imi_cuda_page_write_args a;
    int shift, cpr;   // log2(page); 8-element pieces per row (n_head_kv * head_dim / 8)
};

template <typename D> __device__ __forceinline__ D to_page(float x);
template <> __device__ __forceinline__ __half to_page<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 to_page<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// eight elements of a row as the pages' type: S float is rounded once, to nearest even; S == D is copied
template <typename S, typename D, bool VEC>
__device__ __forceinline__ uint4 piece(const S *p) {
    union { D h[8]; uint4 u; } o;
    if constexpr (sizeof(S) == 4) {
        float f[8];
        if constexpr (VEC) {
            const float4 x = __ldcs((const float4 *) p), y = __ldcs((const float4 *) p + 1);
            f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w; f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) f[k] = p[k];
        }
#pragma unroll
        for (int k = 0; k < 8; k++) o.h[k] = to_page<D>(f[k]);
    } else if constexpr (VEC) {
        o.u = __ldcs((const uint4 *) p);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) o.h[k] = p[k];
    }
    return o.u;
}

// One thread per 16 bytes of a row's head in the pages, for K and V. Bound by HBM: every byte is read once and written
// once: 16,000 rows of 8 heads of 128 in 24.1 us, 5.4 TB/s. Two pieces per thread: 23.7, and 2.3 us against 1.7 for 64 rows.
template <typename S, typename D, bool VEC>
__global__ void __launch_bounds__(256) k_page_write(const __grid_constant__ WriteArgs w) {
    const imi_cuda_page_write_args &a = w.a;
    pdl_wait();
    pdl_trigger();
    const long long i = blockIdx.x * 256LL + threadIdx.x, total = (long long) a.rows * w.cpr;
    if (i >= total) return;
    const int r = (int) (i / w.cpr), c = (int) (i - (long long) r * w.cpr), cph = a.head_dim >> 3, h = c / cph, x = (c - h * cph) << 3;
    const int slot = a.slots[r];
    if (slot < 0) return;
    const int pg = slot >> w.shift;
    if (pg >= a.n_pages) {
        if (a.status) atomicMax(a.status, IMI_DEV_PAGE);
        return;
    }
    const long long src = r * a.row_stride + h * a.head_stride + x;
    const long long dst = (((long long) pg * a.n_head_kv + h) * a.page + (slot & (a.page - 1))) * a.head_dim + x;
    const uint4 k = piece<S, D, VEC>((const S *) a.k + src), v = piece<S, D, VEC>((const S *) a.v + src);
    *(uint4 *) ((D *) a.k_pages + dst) = k;
    *(uint4 *) ((D *) a.v_pages + dst) = v;
}

template <typename S, typename D>
const void *write_fn(bool vec) {
    return vec ? (const void *) k_page_write<S, D, true> : (const void *) k_page_write<S, D, false>;
}

SmemLimit g_map_limit;

}  // namespace
}  // namespace imi

using namespace imi;

extern "C" imi_cuda_status imi_cuda_page_map(int device, const imi_cuda_page_map_args *a, void *stream) {
    if (!a || !a->held || !a->add || !a->table || !a->n_free || !a->start || !a->length || !a->n_free_out || !a->status)
        return set_error(IMI_E_ARG, "page_map: null argument");
    if (a->n < 1 || a->n > MAP_ROWS) return set_error(IMI_E_ARG, "page_map: 1.." + std::to_string(MAP_ROWS) + " requests");
    if (!page_ok(a->page)) return set_error(IMI_E_ARG, "page_map: page must be a power of two, 16..256");
    if (a->n_pages < 1 || (int64_t) a->n_pages * a->page > INT32_MAX)
        return set_error(IMI_E_ARG, "page_map: n_pages * page must fit 31 bits");
    if (a->width < 1 || (int64_t) a->width * a->page > INT32_MAX || a->table_stride < a->width)
        return set_error(IMI_E_ARG, "page_map: bad table width or stride");
    if (a->cap < 0 || (a->cap > 0 && (!a->slots || !a->pos))) return set_error(IMI_E_ARG, "page_map: bad slot arrays");
    if (a->free_cap < 0 || (a->free_cap > 0 && !a->free_pages)) return set_error(IMI_E_ARG, "page_map: bad free list");
    if (a->pos0 < 0 || (int64_t) a->pos0 + (int64_t) a->width * a->page > INT32_MAX)
        return set_error(IMI_E_ARG, "page_map: positions must fit 31 bits");
    for (const void *p : { (const void *) a->held, (const void *) a->add, (const void *) a->table, (const void *) a->free_pages,
                           (const void *) a->n_free, (const void *) a->start, (const void *) a->length, (const void *) a->slots,
                           (const void *) a->pos, (const void *) a->n_free_out, (const void *) a->status })
        if (!aligned(p, 4)) return set_error(IMI_E_ARG, "page_map: a buffer is not 4-byte aligned");
    OnDevice on(device);
    if (!on.ok()) return set_error(IMI_E_NODEV, "no CUDA device " + std::to_string(device));
    if (!all_on_device({ a->held, a->add, a->table, a->free_pages, a->n_free, a->start, a->length, a->slots, a->pos,
                         a->n_free_out, a->status }, device))
        return set_error(IMI_E_ARG, "page_map: every buffer must be device memory of device " + std::to_string(device));
    cudaError_t r = g_map_limit.raise(device, { (const void *) k_page_map }, (3 * MAP_ROWS + 1) * 4);
    if (r == cudaSuccess) {
        MapArgs m = { *a, log2i(a->page) };
        // 2,048 slots per CTA (one pass of four per thread), at most two CTAs per SM's worth
        const int grid = std::max(1, std::min(296, (a->cap + 4 * MAP_THREADS - 1) / (4 * MAP_THREADS)));
        void *args[] = { &m };
        r = launch_pdl((const void *) k_page_map, dim3(grid), MAP_THREADS, (size_t) (3 * a->n + 1) * 4, (cudaStream_t) stream, args);
    }
    if (r != cudaSuccess) return set_error(IMI_E_CUDA, std::string("page_map: ") + cudaGetErrorString(r));
    return IMI_OK;
}

extern "C" imi_cuda_status imi_cuda_page_write(int device, const imi_cuda_page_write_args *a, void *stream) {
    if (!a || a->rows < 0) return set_error(IMI_E_ARG, "page_write: bad arguments");
    if (a->page_type != IMI_F16 && a->page_type != IMI_BF16)
        return set_error(IMI_E_ARG, "page_write: pages are IMI_F16 or IMI_BF16");
    if (a->type != IMI_F32 && a->type != a->page_type)
        return set_error(IMI_E_ARG, "page_write: rows are IMI_F32 or of the pages' type");
    if (a->n_head_kv < 1 || a->n_head_kv > 1024 || a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8)
        return set_error(IMI_E_ARG, "page_write: head_dim a multiple of 8 up to 256, 1..1024 heads");
    if (!page_ok(a->page) || a->n_pages < 1 || (int64_t) a->n_pages * a->page > INT32_MAX)
        return set_error(IMI_E_ARG, "page_write: page must be a power of two, 16..256, and n_pages * page fit 31 bits");
    const int size = a->type == IMI_F32 ? 4 : 2;
    if (a->rows && (!a->k || !a->v || !a->slots || !a->k_pages || !a->v_pages))
        return set_error(IMI_E_ARG, "page_write: null argument");
    if (a->row_stride < 0 || a->head_stride < 0) return set_error(IMI_E_ARG, "page_write: negative stride");
    if (!aligned(a->k, size) || !aligned(a->v, size) || !aligned(a->slots, 4) || !aligned(a->status, 4) ||
        !aligned(a->k_pages, 16) || !aligned(a->v_pages, 16))
        return set_error(IMI_E_ARG, "page_write: a buffer is not aligned (pages: 16 bytes)");
    const int cpr = a->n_head_kv * (a->head_dim / 8);
    const long long blocks = ((long long) a->rows * cpr + 255) / 256;
    if (blocks > INT32_MAX) return set_error(IMI_E_ARG, "page_write: too many rows");
    OnDevice on(device);
    if (!on.ok()) return set_error(IMI_E_NODEV, "no CUDA device " + std::to_string(device));
    if (!all_on_device({ a->k, a->v, a->slots, a->k_pages, a->v_pages, a->status }, device))
        return set_error(IMI_E_ARG, "page_write: every buffer must be device memory of device " + std::to_string(device));
    if (!a->rows) return IMI_OK;
    const bool vec = aligned(a->k, 16) && aligned(a->v, 16) && a->row_stride * size % 16 == 0 && a->head_stride * size % 16 == 0;
    const bool h = a->page_type == IMI_F16;
    const void *fn = a->type == IMI_F32 ? (h ? write_fn<float, __half>(vec) : write_fn<float, __nv_bfloat16>(vec))
                                        : (h ? write_fn<__half, __half>(vec) : write_fn<__nv_bfloat16, __nv_bfloat16>(vec));
    WriteArgs w = { *a, log2i(a->page), cpr };
    void *args[] = { &w };
    const cudaError_t r = launch_pdl(fn, dim3((unsigned) blocks), 256, 0, (cudaStream_t) stream, args);
    if (r != cudaSuccess) return set_error(IMI_E_CUDA, std::string("page_write: ") + cudaGetErrorString(r));
    return IMI_OK;
}
