// Attention of one new token per conversation over a shared prompt and the conversation's own pages
// (imi_cuda_prefix_attn).
//
// For a query row (conversation i, head h) with scores s_j = scale q . K_j over the positions it sees,
//     out = sum_j 2^(s_j log2 e - m) V_j / l,   l = sum_j 2^(s_j log2 e - m),   lse = (m + log2 l) / log2 e,
// for any m; a pass keeps m as the running maximum (online softmax), so a list of positions can be cut anywhere: each
// piece gives (m, l, sum) and pieces join by rescaling to the largest m. The shared prompt is cut into pieces that
// serve all conversations at once (rows of many conversations against one read of K and V); each conversation's own
// positions into pieces of equal length; k_join adds them up.
// Scores, maxima, sums and O are held in 32 bits. The weights 2^(s - m) are rounded to the pages' type for their product with V,
// which the matrix instructions take in one type: half a step of it relative to each weight, and l is summed before that rounding.
#include "common.cuh"
#include "serve.h"

#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>

namespace imi {
namespace {

constexpr int PA_ROWS = 4096;             // conversations at most
constexpr int PA_WARPS = 4;               // warps of a piece's CTA
constexpr int PA_STEP = 16;               // positions of a warp's step (a page holds whole steps)
constexpr int PA_POSITIONS = 1 << 30;     // of the prompt and a table row together at most: a position and a piece's length behind it,
                                          // or a whole tile, still fit 32 bits, as do the steps of all rows' tables (pa_shape_ok)
constexpr int PA_MIN_STEPS = 2 * PA_WARPS;   // steps of a piece of the prompt at least
constexpr int PO_MIN_STEPS = 4;           // of an own piece, which is one warp's
constexpr int PO_ITEM_COST = 4, PO_ROUNDS = 3;   // own_plan
constexpr int PO_CTAS(int d) { return d == 64 ? 592 : 296; }   // own CTAs: as many as 148 SMs hold (4 and 2: registers)
constexpr int PA_PRE_ITEMS = 592;         // (row tile, kv head, piece) items aimed at for the prompt: 148 SMs x 4
constexpr int PA_DIRECT = 1024;           // positions (prompt and own) up to which one CTA takes a row alone, per wave of
constexpr int PA_DIRECT_CTAS(int d) { return d == 64 ? 296 : 148; }   // so many (row, kv head)s
constexpr int PA_DWARPS = 8;              // its warps
constexpr int JOIN_WARPS = 148 * 4 * 8;   // of k_join<, 4>, that the SMs hold at once (registers)

struct PaArgs {
    imi_cuda_prefix_attn_args a;
    int shift, g;               // log2(page); heads per kv head
    float sl2;                  // scale * log2(e)
    int pre_splits, pre_len;    // pieces of the prompt and their positions
    float *po;                  // pieces' sums [slot][head_dim]: prompt slots (row * n_head + head) * pre_splits + piece,
    float2 *pml;                // then own slots (off[row] + piece) * n_head + head; (m, l) per slot
    int own_slot0;              // the first own slot
    int *off;                   // own pieces in front of each row [rows + 1]
    // the prompt on the 5th-generation tensor cores (k_pa_mma): units of PM_ROWS query rows of a kv head, `tiles` position
    // tiles each, `span` apart in one line cut every `per` tiles; pair: both streams of a CTA on one row tile
    bool mma, pair;
    int tiles, span, per, rtiles;
};

template <typename T> struct Half2;
template <> struct Half2<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *(const uint32_t *) &h;
    }
    static __device__ __forceinline__ uint32_t times_zero(uint32_t x) {   // what is not finite becomes NaN
        const __half2 h = __hmul2(*(const __half2 *) &x, __floats2half2_rn(0.0f, 0.0f));
        return *(const uint32_t *) &h;
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Half2<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *(const uint32_t *) &h;
    }
    static __device__ __forceinline__ uint32_t times_zero(uint32_t x) {   // what is not finite becomes NaN
        const __nv_bfloat162 h = __hmul2(*(const __nv_bfloat162 *) &x, __floats2bfloat162_rn(0.0f, 0.0f));
        return *(const uint32_t *) &h;
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint4 ldg16(const void *p) { return __ldg((const uint4 *) p); }

template <typename O> __device__ __forceinline__ void put4(O *p, float4 v);
template <> __device__ __forceinline__ void put4<float>(float *p, float4 v) { *(float4 *) p = v; }
template <> __device__ __forceinline__ void put4<__half>(__half *p, float4 v) {
    *(uint2 *) p = make_uint2(Half2<__half>::pack(v.x, v.y), Half2<__half>::pack(v.z, v.w));
}
template <> __device__ __forceinline__ void put4<__nv_bfloat16>(__nv_bfloat16 *p, float4 v) {
    *(uint2 *) p = make_uint2(Half2<__nv_bfloat16>::pack(v.x, v.y), Half2<__nv_bfloat16>::pack(v.z, v.w));
}
__device__ __forceinline__ void put_out(const imi_cuda_prefix_attn_args &a, long long at, float4 v) {
    if (a.out_type == IMI_F32) put4((float *) a.out + at, v);
    else if (a.out_type == IMI_F16) put4((__half *) a.out + at, v);
    else put4((__nv_bfloat16 *) a.out + at, v);
}

// the positions of conversation i that its query sees: the prompt's from `plo`, its own from `olo` to `len`. A row that is not in
// use (len negative) sees nothing, so that under a window it does not hold down what the rows beside it are read from
struct Seen {
    int len, plo, olo;
};
__device__ __forceinline__ Seen seen_of(const PaArgs &p, int i) {
    const imi_cuda_prefix_attn_args &a = p.a;
    int len = a.length[i];
    const int cap = a.width << p.shift;
    if (len > cap) {
        if (a.status) atomicMax(a.status, IMI_DEV_TABLE);
        len = cap;
    }
    if (len < 0) return { len, a.prefix_len, 0 };
    const int low = a.window > 0 ? max(0, a.prefix_len + len - a.window) : 0;
    return { len, min(low, a.prefix_len), max(0, low - a.prefix_len) };
}

// ---- a warp's pass over 16 query rows: matrix instructions on registers alone ----
// m16n8k16 sums over k in any order, so K is read as the lanes can load it: lane (n = lane / 4, t = lane % 4) takes
// whole 16-byte pieces 8t..8t+7 (+32, ..) of position n's row, and the query's operand uses the same order. V needs two
// positions of one dimension in a register: lane (w = lane / 4, t) loads the 16 bytes 8w..8w+7 of positions 2t, 2t+1,
// 2t+8, 2t+9 and pairs them with byte permutes; product j then holds dimension 8n + j at its column n. Nothing passes
// through shared memory. R8: at most 8 query rows (the fragment's upper rows are zero and not kept).
constexpr int PO_STAGES = 3;              // steps of own positions in a warp's ring

template <typename T, int D, bool R8>
struct Pass {
    static constexpr int KC = D / 32, NO = D / 8, HV = D / 64, RH = R8 ? 2 : 4;
    uint32_t q[D / 16][R8 ? 2 : 4];
    float o[NO][RH];
    float m0, m1, l0, l1;

    __device__ __forceinline__ void init() {
#pragma unroll
        for (int j = 0; j < NO; j++)
#pragma unroll
            for (int e = 0; e < RH; e++) o[j][e] = 0.0f;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.0f;
    }
    // the query's operand: qr0, qr1 the rows of this lane (null: zeros)
    __device__ __forceinline__ void load_q(const T *qr0, const T *qr1) {
        const int t = threadIdx.x & 3;
#pragma unroll
        for (int c = 0; c < KC; c++) {
            uint4 x = make_uint4(0, 0, 0, 0), y = x;
            if (qr0) x = ldg16(qr0 + 32 * c + 8 * t);
            if (!R8 && qr1) y = ldg16(qr1 + 32 * c + 8 * t);
            if constexpr (R8) {
                q[2 * c][0] = x.x; q[2 * c][1] = x.y; q[2 * c + 1][0] = x.z; q[2 * c + 1][1] = x.w;
            } else {
                q[2 * c][0] = x.x; q[2 * c][1] = y.x; q[2 * c][2] = x.y; q[2 * c][3] = y.y;
                q[2 * c + 1][0] = x.z; q[2 * c + 1][1] = y.z; q[2 * c + 1][2] = x.w; q[2 * c + 1][3] = y.w;
            }
        }
    }
    // a step's scores c (8 positions x 2, this lane's rows) into probabilities, the running maximum and sums with them
    __device__ __forceinline__ void soft(float (&c)[2][4], uint32_t (&pa)[4]) {
        float x0 = fmaxf(fmaxf(c[0][0], c[0][1]), fmaxf(c[1][0], c[1][1]));
        x0 = fmaxf(x0, __shfl_xor_sync(~0u, x0, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(~0u, x0, 2));
        const float n0 = fmaxf(m0, x0);
        float n1 = -INFINITY;
        if constexpr (!R8) {
            float x1 = fmaxf(fmaxf(c[0][2], c[0][3]), fmaxf(c[1][2], c[1][3]));
            x1 = fmaxf(x1, __shfl_xor_sync(~0u, x1, 1));
            x1 = fmaxf(x1, __shfl_xor_sync(~0u, x1, 2));
            n1 = fmaxf(m1, x1);
        }
        const float u0 = n0 == -INFINITY ? 0.0f : n0, u1 = n1 == -INFINITY ? 0.0f : n1;
        if (__any_sync(~0u, n0 != m0 || (!R8 && n1 != m1))) {
            const float f0 = ex2(m0 - u0), f1 = R8 ? 1.0f : ex2(m1 - u1);
            l0 *= f0;
            l1 *= f1;
#pragma unroll
            for (int j = 0; j < NO; j++) {
                o[j][0] *= f0; o[j][1] *= f0;
                if constexpr (!R8) { o[j][2] *= f1; o[j][3] *= f1; }
            }
            m0 = n0;
            m1 = n1;
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float e0 = ex2(c[i][0] - u0), e1 = ex2(c[i][1] - u0);
            l0 += e0 + e1;
            pa[2 * i] = Half2<T>::pack(e0, e1);
            if constexpr (R8) pa[2 * i + 1] = 0;
            else {
                const float e2 = ex2(c[i][2] - u1), e3 = ex2(c[i][3] - u1);
                l1 += e2 + e3;
                pa[2 * i + 1] = Half2<T>::pack(e2, e3);
            }
        }
    }
    // scores in powers of two; positions outside [lo0 or lo1, hi) masked (`none`: all)
    __device__ __forceinline__ void mask(float (&c)[2][4], float sl2, int base, int lo0, int lo1, int hi, bool none) {
        const int t = threadIdx.x & 3;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < RH; e++) c[i][e] *= sl2;
        if (base < lo0 || base < lo1 || base + PA_STEP > hi || none) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < RH; e++) {
                    const int at = base + 8 * i + 2 * t + (e & 1);
                    if (none || at >= hi || at < (e < 2 ? lo0 : lo1)) c[i][e] = -INFINITY;
                }
        }
    }
    // scores of 8 positions, whose K rows this lane holds in 16-byte pieces
    __device__ __forceinline__ void score(float (&c)[4], const uint4 (&kr)[KC]) {
        c[0] = c[1] = c[2] = c[3] = 0.0f;
#pragma unroll
        for (int j = 0; j < KC; j++) {
            const uint4 k = kr[j];
            uint32_t a0[4], a1[4];
            if constexpr (R8) {
                a0[0] = q[2 * j][0]; a0[1] = 0; a0[2] = q[2 * j][1]; a0[3] = 0;
                a1[0] = q[2 * j + 1][0]; a1[1] = 0; a1[2] = q[2 * j + 1][1]; a1[3] = 0;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) { a0[e] = q[2 * j][e]; a1[e] = q[2 * j + 1][e]; }
            }
            Half2<T>::mma(c, a0, k.x, k.y);
            Half2<T>::mma(c, a1, k.z, k.w);
        }
    }
    // sums += P V for a 64-dimension part: vr are this lane's pieces of positions 2t, 2t + 1, 2t + 8, 2t + 9
    __device__ __forceinline__ void add(int h, const uint32_t (&pa)[4], const uint4 (&vr)[4]) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t a = (&vr[0].x)[e], b = (&vr[1].x)[e], c = (&vr[2].x)[e], d = (&vr[3].x)[e];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint32_t sel = k ? 0x7632u : 0x5410u, b0 = __byte_perm(a, b, sel), b1 = __byte_perm(c, d, sel);
                float (&x)[RH] = o[8 * h + 2 * e + k];
                if constexpr (R8) {
                    float y[4] = { x[0], x[1], 0.0f, 0.0f };
                    Half2<T>::mma(y, pa, b0, b1);
                    x[0] = y[0];
                    x[1] = y[1];
                } else {
                    Half2<T>::mma(x, pa, b0, b1);
                }
            }
        }
    }
    // positions [lo, hi) of the pages `list`, steps first, first + stride, .. of 16 positions; lo0, lo1: what this
    // lane's rows see from (>= lo); kb, vb: the kv head's rows in page 0; ps: elements from page to page
    __device__ void run(const PaArgs &p, const int32_t *list, const T *kb, const T *vb, long long ps, int lo, int hi, int lo0,
                        int lo1, int first, int stride) {
        const int lane = threadIdx.x & 31, w = lane >> 2, t = lane & 3, end = (hi + PA_STEP - 1) / PA_STEP;
        int s = lo / PA_STEP + first;
        if (s >= end || lo >= hi) return;
        auto page_at = [&](int step) {
            const int id = step < end ? __ldg(list + (step * PA_STEP >> p.shift)) : 0;
            if ((unsigned) id < (unsigned) p.a.n_pages) return id;
            if (p.a.status) atomicMax(p.a.status, IMI_DEV_PAGE);
            return -1;
        };
        uint4 kr[2][KC];
        auto load_k = [&](int step, int id) {
            if (id < 0) id = 0;   // a page that does not exist: page 0 is read and masked
            const T *r = kb + id * ps + (long long) ((step * PA_STEP & (p.a.page - 1)) + w) * D + 8 * t;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int c = 0; c < KC; c++) kr[i][c] = ldg16(r + 8 * i * D + 32 * c);
        };
        int id = page_at(s);
        load_k(s, id);
        int id1 = page_at(s + stride);
        for (; s < end; s += stride) {
            // this step's V on its way while the scores are made
            uint4 vr[4][HV];
            {
                const T *r = vb + max(id, 0) * ps + (long long) ((s * PA_STEP & (p.a.page - 1)) + 2 * t) * D + 8 * w;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int h = 0; h < HV; h++) vr[i][h] = ldg16(r + ((i & 1) + 8 * (i >> 1)) * D + 64 * h);
            }
            float c[2][4];
            score(c[0], kr[0]);
            score(c[1], kr[1]);
            const int base = s * PA_STEP, id_now = id;
            id = id1;
            if (s + stride < end) load_k(s + stride, id);
            id1 = page_at(s + 2 * stride);
            mask(c, p.sl2, base, lo0, lo1, hi, id_now < 0);
            if (base < lo || base + PA_STEP > hi || id_now < 0)
#pragma unroll
                for (int i = 0; i < 4; i++) {   // what no row sees may be anything: 0 x NaN must not reach the sums
                    const int at = base + 2 * t + (i & 1) + 8 * (i >> 1);
                    if (at < lo || at >= hi || id_now < 0)
#pragma unroll
                        for (int h = 0; h < HV; h++) vr[i][h] = make_uint4(0, 0, 0, 0);
                }
            uint32_t pa[4];
            soft(c, pa);
#pragma unroll
            for (int h = 0; h < HV; h++) {
                const uint4 v[4] = { vr[0][h], vr[1][h], vr[2][h], vr[3][h] };
                add(h, pa, v);
            }
        }
    }
    // the same for a long list of one warp, K and V through a ring of PO_STAGES steps in the warp's shared memory, PO_STAGES - 1 of
    // them on their way: more bytes in flight than registers hold. 16-byte pieces of a row lie at piece ^ x(row), so that neither
    // the copies, nor the eight lanes that read K (two rows, four pieces) or V (four rows, two pieces) at once meet in a bank. Lane
    // w takes V's piece w / 2 + 4 (w % 2): product j then holds dimension 8 t + 32 n + j (+ 64 h) at column 2t + n.
    static constexpr int STAGE = 2 * PA_STEP * D * 2;
    static __device__ __forceinline__ uint32_t place(int row, int piece) {
        return row * (D * 2) + ((piece ^ ((row & 1) << 2 | (row >> 1 & 3))) << 4);
    }
    __device__ void run_ring(const PaArgs &p, uint8_t *ring, const int32_t *list, const T *kb, const T *vb, long long ps, int lo, int hi) {
        const int lane = threadIdx.x & 31, w = lane >> 2, t = lane & 3, end = (hi + PA_STEP - 1) / PA_STEP, s0 = lo / PA_STEP;
        if (lo >= hi) return;
        auto page_at = [&](int step) {
            const int id = step < end ? __ldg(list + (step * PA_STEP >> p.shift)) : 0;
            if ((unsigned) id < (unsigned) p.a.n_pages) return id;
            if (p.a.status) atomicMax(p.a.status, IMI_DEV_PAGE);
            return -1;
        };
        constexpr int CH = D / 8, RP = 32 / CH;   // pieces of a row, rows that a warp copies at once
        const int cr = lane / CH, cc = lane % CH;
        const uint32_t at = smem_u32(ring);
        auto copy = [&](int step, int id) {       // rows that nobody sees, and those of a page that does not exist, as zeros
            if (step < end) {
                const long long off = max(id, 0) * ps + (long long) (step * PA_STEP & (p.a.page - 1)) * D + 8 * cc;
                const uint32_t dst = at + (step - s0) % PO_STAGES * STAGE;
#pragma unroll
                for (int i = 0; i < PA_STEP / RP; i++) {
                    const int row = cr + i * RP, pos = step * PA_STEP + row, bytes = id >= 0 && pos >= lo && pos < hi ? 16 : 0;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + place(row, cc)), "l"(kb + off + row * D), "r"(bytes) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + STAGE / 2 + place(row, cc)), "l"(vb + off + row * D), "r"(bytes) : "memory");
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int ids[PO_STAGES];                       // of the steps whose copies come next
#pragma unroll
        for (int k = 0; k < PO_STAGES; k++) ids[k] = page_at(s0 + k);
#pragma unroll
        for (int k = 0; k < PO_STAGES - 1; k++) copy(s0 + k, ids[k]);
        int next = ids[PO_STAGES - 1];
        unsigned gone = 0;                        // pages that do not exist, per step, the one at hand in bit 0
#pragma unroll
        for (int k = 0; k < PO_STAGES; k++) gone |= (ids[k] < 0) << k;
        for (int s = s0; s < end; s++) {
            copy(s + PO_STAGES - 1, next);
            next = page_at(s + PO_STAGES);
            asm volatile("cp.async.wait_group %0;" ::"n"(PO_STAGES - 1) : "memory");
            __syncwarp();
            const uint8_t *k = ring + (s - s0) % PO_STAGES * STAGE, *v = k + STAGE / 2;
            float c[2][4];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                uint4 kr[KC];
#pragma unroll
                for (int x = 0; x < KC; x++) kr[x] = *(const uint4 *) (k + place(8 * i + w, 4 * x + t));
                score(c[i], kr);
            }
            mask(c, p.sl2, s * PA_STEP, lo, lo, hi, gone & 1);
            uint32_t pa[4];
            soft(c, pa);
#pragma unroll
            for (int h = 0; h < HV; h++) {
                uint4 vr[4];
#pragma unroll
                for (int i = 0; i < 4; i++) vr[i] = *(const uint4 *) (v + place(2 * t + (i & 1) + 8 * (i >> 1), 8 * h + (w >> 1) + 4 * (w & 1)));
                add(h, pa, vr);
            }
            gone = gone >> 1 | (next < 0) << (PO_STAGES - 1);
            __syncwarp();
        }
    }
    // the sums of the lanes that share a row
    __device__ __forceinline__ void finish() {
        l0 += __shfl_xor_sync(~0u, l0, 1);
        l0 += __shfl_xor_sync(~0u, l0, 2);
        if constexpr (!R8) {
            l1 += __shfl_xor_sync(~0u, l1, 1);
            l1 += __shfl_xor_sync(~0u, l1, 2);
        }
    }
    // this warp's result into shared memory: rows of D + 4 floats (m, l, and padding that spreads the banks, behind)
    __device__ __forceinline__ void put(float *sh) const {
        const int lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
#pragma unroll
        for (int up = 0; up < (R8 ? 1 : 2); up++) {
            float *row = sh + (r + 8 * up) * (D + 4);
#pragma unroll
            for (int h = 0; h < HV; h++)
#pragma unroll
                for (int n = 0; n < 2; n++)   // column n of the products: dimensions 64 h + 8 (2t + n) + 0..7
#pragma unroll
                    for (int j = 0; j < 8; j += 4)
                        *(float4 *) (row + 64 * h + 16 * t + 8 * n + j) =
                            make_float4(o[8 * h + j][2 * up + n], o[8 * h + j + 1][2 * up + n], o[8 * h + j + 2][2 * up + n],
                                        o[8 * h + j + 3][2 * up + n]);
            if (t == 0) {
                row[D] = up ? m1 : m0;
                row[D + 1] = up ? l1 : l0;
            }
        }
    }
};

// the NW warps' results of `rows` query rows joined: four dimensions per thread; emit(row, dimension, sum, m, l)
template <int D, int NW, int ROWS, typename F>
__device__ __forceinline__ void join_warps(const float *sh, int rows, F emit) {
    for (int x = threadIdx.x; x < rows * (D / 4); x += NW * 32) {
        const int r = x / (D / 4), c = x % (D / 4) * 4;
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; k++) m = fmaxf(m, sh[(k * ROWS + r) * (D + 4) + D]);
        const float u = m == -INFINITY ? 0.0f : m;
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < NW; k++) {
            const float *row = sh + (k * ROWS + r) * (D + 4);
            const float f = ex2(row[D] - u);
            const float4 v = *(const float4 *) (row + c);
            l = fmaf(f, row[D + 1], l);
            s.x = fmaf(f, v.x, s.x); s.y = fmaf(f, v.y, s.y); s.z = fmaf(f, v.z, s.z); s.w = fmaf(f, v.w, s.w);
        }
        emit(r, c, s, m, l);
    }
}
__device__ __forceinline__ float4 scaled(float4 s, float l) {
    const float f = l > 0.0f ? __fdiv_rn(1.0f, l) : (l == 0.0f ? 0.0f : l);   // l NaN stays NaN
    return make_float4(s.x * f, s.y * f, s.z * f, s.w * f);
}
constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896340736f;
__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.0f ? -INFINITY : (m + log2f(l)) * LN2; }

// ---- few positions: one CTA per (conversation, kv head) takes all of them, its warps step by step in turn ----
// One launch, no pieces. Bound by its chain of reads: the lengths, page numbers, rows. A whole call against the pieces' launches:
// 1 conversation on 200 positions 4.5 us (8.3), on 1,000 8.4 (8.6), on 2,000 14.3 (8.8); 64 on 400 11.0 (15.9); 256 on 220 31 (20.3).
template <typename T, int D, bool R8>
__global__ void __launch_bounds__(PA_DWARPS * 32) k_pa_direct(const __grid_constant__ PaArgs p) {
    constexpr int ROWS = R8 ? 8 : 16;
    extern __shared__ float shf[];
    const imi_cuda_prefix_attn_args &a = p.a;
    pdl_wait();
    pdl_trigger();
    const int i = blockIdx.x / a.n_head_kv, kvh = blockIdx.x % a.n_head_kv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Seen v = seen_of(p, i);
    if (v.len < 0) return;
    const T *q = (const T *) a.q + i * a.q_stride + (long long) kvh * p.g * D;
    const int r = lane >> 2;
    Pass<T, D, R8> f;
    f.init();
    f.load_q(r < p.g ? q + r * D : nullptr, r + 8 < p.g ? q + (r + 8) * D : nullptr);
    const long long ps = (long long) a.n_head_kv * a.page * D, head = (long long) kvh * a.page * D;
    const T *kb = (const T *) a.k_pages + head, *vb = (const T *) a.v_pages + head;
    f.run(p, a.prefix, kb, vb, ps, v.plo, a.prefix_len, v.plo, v.plo, warp, PA_DWARPS);
    f.run(p, a.table + i * a.table_stride, kb, vb, ps, v.olo, v.len, v.olo, v.olo, PA_DWARPS - 1 - warp, PA_DWARPS);
    f.finish();
    f.put(shf + warp * ROWS * (D + 4));
    __syncthreads();
    join_warps<D, PA_DWARPS, ROWS>(shf, p.g, [&](int row, int c, float4 s, float m, float l) {
        const int h = kvh * p.g + row;
        put_out(a, i * a.out_stride + (long long) h * D + c, scaled(s, l));
        if (c == 0 && a.lse) a.lse[(long long) i * a.n_head + h] = lse_of(m, l);
    });
}

// ---- pieces ----
// own pieces of every row into off[0..rows] (shared memory): steps of 16 positions, `chunk` steps per piece. A warp takes one
// (piece, kv head) item after the other, so the time is rounds x (chunk + what an item costs beside its steps, about
// PO_ITEM_COST). Either a chunk so long that one round does, or PO_ROUNDS rounds of short ones, which the rows' last pieces and
// their different lengths do less harm. Every CTA works this out from the lengths (4 bytes per row from L2). Returns chunk.
__device__ int own_plan(const PaArgs &p, int *off, int *tmp) {
    const imi_cuda_prefix_attn_args &a = p.a;
    const int tid = threadIdx.x, nt = PA_WARPS * 32, lane = tid & 31, warp = tid >> 5;
    const int per = (a.rows + nt - 1) / nt, i0 = min(a.rows, tid * per), i1 = min(a.rows, i0 + per);
    int sum = 0, most = 0, live = 0;
    for (int i = i0; i < i1; i++) {
        const Seen v = seen_of(p, i);
        const int steps = v.len > v.olo ? (v.len + PA_STEP - 1) / PA_STEP - v.olo / PA_STEP : 0;
        off[i + 1] = steps;
        sum += steps;
        most = max(most, steps);
        live += steps > 0;
    }
    sum = __reduce_add_sync(~0u, sum);
    most = __reduce_max_sync(~0u, most);
    live = __reduce_add_sync(~0u, live);
    if (lane == 0) { tmp[3 * warp] = sum; tmp[3 * warp + 1] = most; tmp[3 * warp + 2] = live; }
    __syncthreads();
    sum = most = live = 0;
#pragma unroll
    for (int w = 0; w < PA_WARPS; w++) {
        sum += tmp[3 * w];
        most = max(most, tmp[3 * w + 1]);
        live += tmp[3 * w + 2];
    }
    const long long warps = (long long) gridDim.x * PA_WARPS, work = (long long) sum * a.n_head_kv, rows = (long long) live * a.n_head_kv;
    // one round: at most work / chunk + rows items
    const int one = rows < warps ? (int) min((long long) max(1, most), (work + warps - rows - 1) / (warps - rows)) : INT32_MAX;
    int chunk = max(PO_MIN_STEPS, (int) min((long long) PA_POSITIONS / PA_STEP, (work + PO_ROUNDS * warps - 1) / (PO_ROUNDS * warps)));
    const long long rounds = (work / chunk + rows + warps - 1) / warps;
    if (one < INT32_MAX && one + PO_ITEM_COST <= rounds * (chunk + PO_ITEM_COST)) chunk = max(PO_MIN_STEPS, one);
    int cnt = 0;
    for (int i = i0; i < i1; i++) cnt += (off[i + 1] + chunk - 1) / chunk;
    int at = cnt;   // exclusive sums over the threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(~0u, at, o);
        if (lane >= o) at += z;
    }
    if (lane == 31) tmp[16 + warp] = at;
    __syncthreads();
    at -= cnt;
#pragma unroll
    for (int w = 0; w < PA_WARPS; w++)
        if (w < warp) at += tmp[16 + w];
    for (int i = i0; i < i1; i++) {
        at += (off[i + 1] + chunk - 1) / chunk;
        off[i + 1] = at;
    }
    if (tid == 0) off[0] = 0;
    __syncthreads();
    return chunk;
}

// the prompt for few query rows: CTA items are (piece, tile of 16 query rows, kv head). Bound by the bytes of K and V, which
// every tile of rows reads anew: one conversation on 20,000 positions (47 MB with its own) 20.4 us in all, 2.3 TB/s
template <typename T, int D>
__global__ void __launch_bounds__(PA_WARPS * 32) k_pa_pieces(const __grid_constant__ PaArgs p) {
    constexpr int ROWS = 16;
    extern __shared__ float shf[];
    const imi_cuda_prefix_attn_args &a = p.a;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2;
    const long long ps = (long long) a.n_head_kv * a.page * D;
    const int qrows = a.rows * p.g, tiles = (qrows + ROWS - 1) / ROWS, items = tiles * a.n_head_kv * p.pre_splits;
    for (int it = blockIdx.x; it < items; it += gridDim.x) {
        Pass<T, D, false> f;
        f.init();
        const int kvh = it % a.n_head_kv, k = it / a.n_head_kv, tile = k % tiles, piece = k / tiles, fr0 = tile * ROWS,
                  nr = min(ROWS, qrows - fr0);
        const T *q = (const T *) a.q + (long long) kvh * p.g * D;
        auto qrow = [&](int x) -> const T * {
            if (x >= nr) return nullptr;
            const int fr = fr0 + x;
            return q + fr / p.g * a.q_stride + (long long) (fr % p.g) * D;
        };
        f.load_q(qrow(r), qrow(r + 8));
        const long long head = (long long) kvh * a.page * D;
        int lo0 = 0, lo1 = 0, lo = piece * p.pre_len;
        const int hi = min(a.prefix_len, lo + p.pre_len);
        if (a.window > 0) {
            if (r < nr) lo0 = seen_of(p, (fr0 + r) / p.g).plo;
            if (r + 8 < nr) lo1 = seen_of(p, (fr0 + r + 8) / p.g).plo;
            lo = max(lo, __reduce_min_sync(~0u, min(r < nr ? lo0 : INT32_MAX, r + 8 < nr ? lo1 : INT32_MAX)));
        }
        f.run(p, a.prefix, (const T *) a.k_pages + head, (const T *) a.v_pages + head, ps, lo, hi, lo0, lo1, warp, PA_WARPS);
        f.finish();
        __syncthreads();   // the item before has been read
        f.put(shf + warp * ROWS * (D + 4));
        __syncthreads();
        join_warps<D, PA_WARPS, ROWS>(shf, nr, [&](int x, int c, float4 s, float m, float l) {
            const int fr = fr0 + x, i = fr / p.g, h = kvh * p.g + fr % p.g;
            const long long slot = ((long long) i * a.n_head + h) * p.pre_splits + piece;
            *(float4 *) (p.po + slot * D + c) = s;
            if (c == 0) p.pml[slot] = make_float2(m, l);
        });
    }
}

// the conversations' own positions: a warp's item is a (piece, kv head), its 16-position steps one after the other. Bound by
// HBM: every row of K and V is read once: 65 MB of 64 conversations' in 13.7 us (median CTA; the last one 18.5)
template <typename T, int D, bool R8>
__global__ void __launch_bounds__(PA_WARPS * 32) k_pa_own(const __grid_constant__ PaArgs p) {
    extern __shared__ __align__(128) uint8_t shb[];
    __shared__ int tmp[32];
    int *off = (int *) (shb + PA_WARPS * PO_STAGES * Pass<T, D, R8>::STAGE);
    const imi_cuda_prefix_attn_args &a = p.a;
    // behind a launch for the prompt: that launch has let these CTAs start when all of its own had done their wait, and shares
    // nothing with them; they wait for it at their end, so that k_join, which waits for them, has both
    const bool early = a.prefix_len > 0;
    if (!early) pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, t = lane & 3;
    const long long ps = (long long) a.n_head_kv * a.page * D;
    const int chunk = own_plan(p, off, tmp), items = off[a.rows] * a.n_head_kv;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i <= a.rows; i += PA_WARPS * 32) p.off[i] = off[i];
    for (int it = blockIdx.x * PA_WARPS + warp; it < items; it += gridDim.x * PA_WARPS) {
        const int kvh = it % a.n_head_kv, k = it / a.n_head_kv;
        int row = 0, up = a.rows;   // the row whose pieces hold k
        while (up - row > 1) {
            const int mid = (row + up) >> 1;
            if (off[mid] <= k) row = mid;
            else up = mid;
        }
        const int piece = k - off[row];
        const T *q = (const T *) a.q + row * a.q_stride + (long long) kvh * p.g * D;
        Pass<T, D, R8> f;
        f.init();
        f.load_q(r < p.g ? q + r * D : nullptr, r + 8 < p.g ? q + (r + 8) * D : nullptr);
        const long long head = (long long) kvh * a.page * D;
        const Seen v = seen_of(p, row);
        const int s0 = v.olo / PA_STEP + piece * chunk, lo = max(v.olo, s0 * PA_STEP), hi = (int) min((long long) v.len, (s0 + (long long) chunk) * PA_STEP);
        f.run_ring(p, shb + warp * PO_STAGES * Pass<T, D, R8>::STAGE, a.table + row * a.table_stride, (const T *) a.k_pages + head,
                   (const T *) a.v_pages + head, ps, lo, hi);
        f.finish();
        const long long slot0 = p.own_slot0 + (long long) k * a.n_head + kvh * p.g;
#pragma unroll
        for (int x = 0; x < (R8 ? 1 : 2); x++)
            if (r + 8 * x < p.g) {
                float *o = p.po + (slot0 + r + 8 * x) * D;
#pragma unroll
                for (int h = 0; h < D / 64; h++)
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int j = 0; j < 8; j += 4)
                            *(float4 *) (o + 64 * h + 8 * t + 32 * n + j) =
                                make_float4(f.o[8 * h + j][2 * x + n], f.o[8 * h + j + 1][2 * x + n], f.o[8 * h + j + 2][2 * x + n],
                                            f.o[8 * h + j + 3][2 * x + n]);
                if (t == 0) p.pml[slot0 + r + 8 * x] = make_float2(x ? f.m1 : f.m0, x ? f.l1 : f.l0);
            }
    }
    if (early) pdl_wait();
}

#include "serve_mma.cuh"

// out and lse of every (row, head) from its pieces: `ways` (1, 2, 4 or 8) warps each, UN pieces' values of each on their way.
// Bound by latency: the prompt's first pieces are asked for beside the length and the own pieces' place, not behind them.
template <int D, int UN>
__global__ void __launch_bounds__(256, UN == 2 ? 7 : UN == 4 ? 4 : 2) k_join(const __grid_constant__ PaArgs p, int ways) {
    __shared__ float sh[8][D + 4];
    const imi_cuda_prefix_attn_args &a = p.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, way = warp % ways;
    const int x = blockIdx.x * (8 / ways) + warp / ways, i = x / a.n_head, h = x % a.n_head, ic = min(i, a.rows - 1);
    int np = p.pre_splits;   // the prompt's pieces of this row
    if (p.mma) {
        const int u0 = (h / p.g * p.rtiles + (i * p.g + h % p.g) / (p.pair ? PM_M : PM_ROWS)) * p.span;
        np = ((u0 + p.tiles - 1) / p.per - u0 / p.per + 1) * (p.pair ? 2 : 1);
    }
    if (i >= a.rows) np = 0;
    // D / 4 lanes hold four dimensions each; at D 64 the warp's halves take every other piece
    constexpr int G = 32 / (D / 4);
    const int part = lane / (D / 4), c = lane % (D / 4) * 4, step = G * ways;
    const float *po = p.po + c;
    float2 ml[UN];
    float4 v[UN];
    auto load = [&](int e, long long slot) {
        ml[e] = p.pml[slot];
        v[e] = *(const float4 *) (po + slot * D);
    };
    pdl_wait();
    pdl_trigger();
    const int len = a.length[ic], o0 = p.off[ic], o1 = p.off[ic + 1];
    int k = way * G + part;   // this lane's next piece
#pragma unroll
    for (int e = 0; e < UN; e++)
        if (k + e * step < np) load(e, (long long) x * p.pre_splits + k + e * step);
    const bool live = i < a.rows && len >= 0;
    float m = -INFINITY, l = 0.0f;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (live) {
        const int n = np + o1 - o0;
        const long long own = p.own_slot0 + (long long) (o0 - np) * a.n_head + h;
#pragma unroll
        for (int e = 0; e < UN; e++) {
            const int q = k + e * step;
            if (q >= n) ml[e] = make_float2(-INFINITY, 0.0f);
            else if (q >= np) load(e, own + (long long) q * a.n_head);
        }
        while (true) {
#pragma unroll
            for (int e = 0; e < UN; e++) {
                const float top = fmaxf(m, ml[e].x), u = top == -INFINITY ? 0.0f : top, f = ex2(m - u), g = ex2(ml[e].x - u);
                l = fmaf(l, f, g * ml[e].y);
                // a piece that saw nothing adds nothing, whatever its sums hold
                if (ml[e].x > -INFINITY) {
                    s.x = fmaf(s.x, f, g * v[e].x); s.y = fmaf(s.y, f, g * v[e].y);
                    s.z = fmaf(s.z, f, g * v[e].z); s.w = fmaf(s.w, f, g * v[e].w);
                }
                m = top;
            }
            k += UN * step;
            if (k - part >= n) break;
#pragma unroll
            for (int e = 0; e < UN; e++) {
                const int q = k + e * step;
                if (q < n) load(e, q < np ? (long long) x * p.pre_splits + q : own + (long long) q * a.n_head);
                else ml[e] = make_float2(-INFINITY, 0.0f);
            }
        }
        if (G == 2) {
            const float om = __shfl_xor_sync(~0u, m, 16), top = fmaxf(m, om), u = top == -INFINITY ? 0.0f : top, f = ex2(m - u);
            l *= f;
            s.x *= f; s.y *= f; s.z *= f; s.w *= f;
            l += __shfl_xor_sync(~0u, l, 16);
            s.x += __shfl_xor_sync(~0u, s.x, 16); s.y += __shfl_xor_sync(~0u, s.y, 16);
            s.z += __shfl_xor_sync(~0u, s.z, 16); s.w += __shfl_xor_sync(~0u, s.w, 16);
            m = top;
        }
    }
    if (ways > 1) {
        if (part == 0) *(float4 *) &sh[warp][c] = s;
        if (lane == 0) { sh[warp][D] = m; sh[warp][D + 1] = l; }
        __syncthreads();
        if (way) return;
        for (int w = 1; w < ways; w++) {
            const float *q = sh[warp + w];
            const float4 v = *(const float4 *) (q + c);
            const float om = q[D], top = fmaxf(m, om), u = top == -INFINITY ? 0.0f : top, f = ex2(m - u), g = ex2(om - u);
            l = fmaf(l, f, g * q[D + 1]);
            s.x = fmaf(s.x, f, g * v.x); s.y = fmaf(s.y, f, g * v.y); s.z = fmaf(s.z, f, g * v.z); s.w = fmaf(s.w, f, g * v.w);
            m = top;
        }
    }
    if (!live) return;
    if (part == 0) put_out(a, i * a.out_stride + (long long) h * D + c, scaled(s, l));
    if (lane == 0 && a.lse) a.lse[x] = lse_of(m, l);
}

// ---- host ----
// how a call is cut: pieces of the prompt, slots of the workspace
struct PaPlan {
    int splits, len;        // pieces of a query row over the prompt at most; positions of a piece (k_pa_pieces)
    bool mma, pair;
    int tiles, span, per, rtiles, grid, own_sms;
    size_t pre_slots, own_slots;
    size_t off_bytes, bytes;
};
// The prompt's tiles over `sms` CTAs: either a whole number of pieces per unit, or the line cut evenly, whose CTAs may have to
// begin a unit anew (about PM_BEGIN tiles' time each). Returns the tiles' time of the longest CTA.
int pm_cut(PaPlan &p, int n_head_kv, int sms) {
    const long long units = (long long) p.rtiles * n_head_kv, total = units * p.tiles;
    const long long k = std::max(1ll, std::min<long long>(sms / units, p.tiles)), whole = (p.tiles + k - 1) / k, even = (total + sms - 1) / sms;
    const long long t_whole = (units * k + sms - 1) / sms * (whole + PM_BEGIN), t_even = even + PM_BEGIN * (1 + (even + p.tiles - 1) / p.tiles);
    const bool cut = t_whole > t_even;
    p.per = (int) std::max<long long>(PM_MIN_TILES, std::min<long long>(PM_MAX_TILES, cut ? even : whole));
    p.span = cut ? p.tiles : (p.tiles + p.per - 1) / p.per * p.per;
    p.grid = (int) ((units * p.span + p.per - 1) / p.per);
    p.splits = ((p.tiles + p.per - 1) / p.per + (cut ? 1 : 0)) * (p.pair ? 2 : 1);
    return (int) std::min<long long>(INT32_MAX, std::max<long long>(std::min(t_whole, t_even), p.per + PM_BEGIN));
}

// own_most: own positions of a row at most
PaPlan pa_plan(int rows, int n_head, int n_head_kv, int head_dim, int prefix_len, long long own_most) {
    PaPlan p = {};
    p.own_sms = 148;
    const int g = n_head / n_head_kv, R = 16, tiles = (rows * g + R - 1) / R;
    p.mma = rows * g > PM_MIN_ROWS && prefix_len > 0;
    if (p.mma) {
        p.pair = rows * g <= PM_M;
        p.rtiles = p.pair ? 1 : (rows * g + PM_ROWS - 1) / PM_ROWS;
        p.tiles = (prefix_len + PM_N - 1) / PM_N;
        // The prompt's CTAs take a whole SM each, and wait for their exponentials; the own positions wait for HBM. So both run at
        // once where that is shorter than one after the other, the own ones, taken to be half of what the tables hold, on the SMs
        // that are left (45 GB/s each). They may be fewer: the prompt is not made slower than by a quarter (and 4 us) for them.
        // 256 conversations on 16,384 positions with 128 own ones each: 81 us one after the other, 77 at once; 64 on 8,000 with 50: 28, 23.5
        const double tile = head_dim == 64 ? 1.55 : 1.9, begin = 5.0;
        const double own = 2.0 * rows * n_head_kv * head_dim * (double) own_most / 45e3;
        const double alone = begin + tile * pm_cut(p, n_head_kv, 148);
        double best = own_most ? alone + 3.0 + own / 148 : alone;
        int sms = 148;
        for (int x = 144; x >= 8 && own_most; x -= 4) {
            const double t = begin + tile * pm_cut(p, n_head_kv, x), o = 3.0 + own / (148 - x);
            if (t > 1.25 * alone + 4.0) break;
            if (std::max(t, o) < best) {
                best = std::max(t, o);
                sms = x;
            }
        }
        pm_cut(p, n_head_kv, sms);
        if (p.grid <= sms && sms < 148) p.own_sms = 148 - p.grid;
    }
    const int steps = (prefix_len + PA_STEP - 1) / PA_STEP;
    if (!p.mma) p.splits = prefix_len ? std::max(1, std::min(PA_PRE_ITEMS / std::max(1, tiles * n_head_kv), steps / PA_MIN_STEPS)) : 0;
    if (p.splits && !p.mma) {
        p.len = (steps + p.splits - 1) / p.splits * PA_STEP;
        p.splits = (prefix_len + p.len - 1) / p.len;
    }
    // slots for the prompt's pieces: at most this many for any call of no more rows and positions, so that its workspace serves
    // them. k_pa_mma: 148 CTAs' pieces of PM_ROWS rows, and up to 3 more pieces (those that PM_MAX_TILES ends besides) of every
    // unit; k_pa_pieces: its items' rows, and one piece of every row
    const size_t units = (size_t) ((rows * g + PM_ROWS - 1) / PM_ROWS) * n_head_kv, most_tiles = ((size_t) prefix_len + PM_N - 1) / PM_N;
    p.pre_slots = prefix_len ? std::max((size_t) PM_ROWS * (148 + units * (3 + most_tiles / PM_MAX_TILES)),
                                        (size_t) R * PA_PRE_ITEMS + (size_t) tiles * R * n_head_kv)
                             : 0;
    p.own_slots = ((size_t) rows + (PO_ROUNDS * PO_CTAS(head_dim) * PA_WARPS + n_head_kv - 1) / n_head_kv) * n_head;
    p.off_bytes = ((size_t) (rows + 1) * 4 + 255) / 256 * 256;
    const size_t slots = p.pre_slots + p.own_slots;
    p.bytes = p.off_bytes + (slots * 8 + 255) / 256 * 256 + slots * head_dim * 4;
    return p;
}

bool pa_shape_ok(int rows, int n_head, int n_head_kv, int head_dim, int prefix_len, int width, int page) {
    return rows >= 0 && rows <= PA_ROWS && n_head_kv >= 1 && n_head >= n_head_kv && n_head <= 1024 && n_head % n_head_kv == 0 &&
           n_head / n_head_kv <= 16 && (head_dim == 64 || head_dim == 128) && prefix_len >= 0 && width >= 0 && page_ok(page) &&
           (int64_t) width * page + prefix_len + page <= PA_POSITIONS && (int64_t) width * page / PA_STEP * rows <= INT32_MAX;
}

// the pages of K (or V) as rows of head_dim values, copied in boxes of up to 128 rows x 64 values with the 128-byte swizzle
cudaError_t page_map_of(const imi_cuda_prefix_attn_args &a, const void *pages, CUtensorMap *out) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    static std::mutex mu;
    {
        std::lock_guard<std::mutex> g(mu);
        if (!encode) {
            void *fn = nullptr;
            cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
            const cudaError_t r = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q);
            if (r != cudaSuccess) return r;
            if (q != cudaDriverEntryPointSuccess || !fn) return cudaErrorNotSupported;
            encode = (PFN_cuTensorMapEncodeTiled_v12000) fn;
        }
    }
    const cuuint64_t dims[2] = { (cuuint64_t) a.head_dim, (cuuint64_t) a.n_pages * a.n_head_kv * a.page },
                     strides[1] = { (cuuint64_t) a.head_dim * 2 };
    const cuuint32_t box[2] = { 64, (cuuint32_t) std::min(a.page, PM_N) }, es[2] = { 1, 1 };
    const CUresult c = encode(out, a.type == IMI_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                              (void *) pages, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return c == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <typename T, int D, bool R8>
cudaError_t launch_pa(PaArgs &p, const PaPlan &pl, cudaStream_t st) {
    const imi_cuda_prefix_attn_args &a = p.a;
    constexpr int ROWS = R8 ? 8 : 16;
    void *args[] = { &p };
    const long long most = (long long) a.prefix_len + ((long long) a.width << p.shift);
    if (most * ((a.rows * a.n_head_kv + PA_DIRECT_CTAS(D) - 1) / PA_DIRECT_CTAS(D)) <= PA_DIRECT)
        return launch_pdl((const void *) k_pa_direct<T, D, R8>, dim3(a.rows * a.n_head_kv), PA_DWARPS * 32,
                          (size_t) PA_DWARPS * ROWS * (D + 4) * 4, st, args);
    cudaError_t r = cudaSuccess;
    if (pl.mma) {
        CUtensorMap km, vm;
        if ((r = page_map_of(a, a.k_pages, &km)) != cudaSuccess || (r = page_map_of(a, a.v_pages, &vm)) != cudaSuccess) return r;
        void *margs[] = { &p, &km, &vm };
        r = launch_pdl((const void *) k_pa_mma<T, D>, dim3(pl.grid), PM_THREADS, PmSmem<D>::TOTAL + 1024, st, margs);
    } else if (pl.splits) {
        const int items = (a.rows * p.g + 15) / 16 * a.n_head_kv * pl.splits;
        r = launch_pdl((const void *) k_pa_pieces<T, D>, dim3(std::min(items, 148 * 16)), PA_WARPS * 32,
                       (size_t) PA_WARPS * 16 * (D + 4) * 4, st, args);
    }
    if (r == cudaSuccess)
        r = launch_pdl((const void *) k_pa_own<T, D, R8>, dim3(PO_CTAS(D) / 148 * pl.own_sms), PA_WARPS * 32, (size_t) PA_WARPS * PO_STAGES * Pass<T, D, R8>::STAGE + (a.rows + 1) * 4, st, args);
    if (r == cudaSuccess) {
        // warps per (row, head): more while a row's pieces (the prompt's, and about a row's share of the own ones) are not asked
        // for all at once and the SMs hold all CTAs at once (a second wave begins 4 us behind the first); then more pieces per
        // warp, where its registers leave one wave too. Where there are more (row, head)s than that, fewer registers for more
        // CTAs per SM. Whole calls: 64 rows of 32 heads 23.6 us with 4 pieces per warp, 31 with 12; 24 of 8, 80 pieces each,
        // 20.6 with 12, 24.4 with 4
        const long long own = 1 + std::min(((long long) a.width << p.shift) / (PO_MIN_STEPS * PA_STEP),
                                           (long long) PO_ROUNDS * PO_CTAS(D) * PA_WARPS / (a.n_head_kv * a.rows));
        const long long all = (long long) a.rows * a.n_head, pieces = pl.splits + own;
        constexpr int G = 128 / D;
        int ways = 1;
        while (ways < 8 && pieces > 4 * G * ways && all * ways * 2 <= JOIN_WARPS) ways *= 2;
        void *jargs[] = { &p, &ways };
        const void *join = all * ways > JOIN_WARPS ? (const void *) k_join<D, 2>
                           : pieces > 4 * G * ways && all * ways <= JOIN_WARPS / 2 ? (const void *) k_join<D, 12>
                                                   : (const void *) k_join<D, 4>;
        r = launch_pdl(join, dim3((unsigned) ((all * ways + 7) / 8)), 256, 0, st, jargs);
    }
    return r;
}
template <typename T>
cudaError_t launch_pa_t(PaArgs &p, const PaPlan &pl, cudaStream_t st) {
    const bool r8 = p.g <= 8;
    if (p.a.head_dim == 64) return r8 ? launch_pa<T, 64, true>(p, pl, st) : launch_pa<T, 64, false>(p, pl, st);
    return r8 ? launch_pa<T, 128, true>(p, pl, st) : launch_pa<T, 128, false>(p, pl, st);
}
template <typename T>
cudaError_t raise_pa(int device) {
    static SmemLimit lim, lim2;
    cudaError_t r = lim.raise(device,
                              { (const void *) k_pa_direct<T, 64, true>, (const void *) k_pa_direct<T, 64, false>,
                                (const void *) k_pa_direct<T, 128, true>, (const void *) k_pa_direct<T, 128, false>,
                                (const void *) k_pa_pieces<T, 64>, (const void *) k_pa_pieces<T, 128>,
                                (const void *) k_pa_own<T, 64, true>, (const void *) k_pa_own<T, 64, false>,
                                (const void *) k_pa_own<T, 128, true>, (const void *) k_pa_own<T, 128, false> },
                              112 * 1024 + PA_ROWS * 4);
    if (r != cudaSuccess) return r;
    r = lim2.raise(device, { (const void *) k_pa_mma<T, 64>, (const void *) k_pa_mma<T, 128> },
                   (int) std::max(PmSmem<64>::TOTAL, PmSmem<128>::TOTAL) + 1024);
    if (r != cudaSuccess) return r;
    static std::atomic<bool> seen{ false };   // a property of the build, the same on every device
    if (seen) return cudaSuccess;
    for (const void *f : { (const void *) k_pa_mma<T, 64>, (const void *) k_pa_mma<T, 128> }) {
        cudaFuncAttributes at;
        if ((r = cudaFuncGetAttributes(&at, f)) != cudaSuccess) return r;
        if (at.numRegs < PM_REGS) return cudaErrorLaunchOutOfResources;
    }
    seen = true;
    return cudaSuccess;
}

}  // namespace
}  // namespace imi

using namespace imi;

extern "C" size_t imi_cuda_prefix_attn_work(int rows, int n_head, int n_head_kv, int head_dim, int prefix_len, int width,
                                            int page) {
    if (!pa_shape_ok(rows, n_head, n_head_kv, head_dim, prefix_len, width, page)) return 0;
    return pa_plan(rows, n_head, n_head_kv, head_dim, prefix_len, (long long) width * page).bytes;
}

extern "C" imi_cuda_status imi_cuda_prefix_attn(int device, const imi_cuda_prefix_attn_args *a, void *stream) {
    if (!a) return set_error(IMI_E_ARG, "prefix_attn: null argument");
    if (a->type != IMI_F16 && a->type != IMI_BF16) return set_error(IMI_E_ARG, "prefix_attn: q and pages are IMI_F16 or IMI_BF16");
    if (a->out_type < IMI_F32 || a->out_type > IMI_BF16) return set_error(IMI_E_ARG, "prefix_attn: bad out_type");
    if (!pa_shape_ok(a->rows, a->n_head, a->n_head_kv, a->head_dim, a->prefix_len, a->width, a->page))
        return set_error(IMI_E_ARG, "prefix_attn: unsupported shape (rows up to " + std::to_string(PA_ROWS) +
                                        ", head_dim 64 or 128, up to 16 heads per kv head, page a power of two in 16..256, prompt and table "
                                        "row below 2^30 positions, all rows' tables below 2^35)");
    if (a->n_pages < 0 || a->window < 0) return set_error(IMI_E_ARG, "prefix_attn: negative n_pages or window");
    if (!std::isfinite(a->scale * LOG2E)) return set_error(IMI_E_ARG, "prefix_attn: scale is not finite, or not in powers of two");
    if (a->rows == 0) return IMI_OK;
    if (((int64_t) a->n_pages * a->n_head_kv + 1) * a->page > INT32_MAX) return set_error(IMI_E_ARG, "prefix_attn: too many pages");
    if ((int64_t) a->rows * a->n_head / PM_ROWS * ((int64_t) a->prefix_len / PM_N + 1) > INT32_MAX / 4)
        return set_error(IMI_E_ARG, "prefix_attn: the prompt is too long for so many rows");
    if (!a->q || !a->out || !a->length || !a->work) return set_error(IMI_E_ARG, "prefix_attn: null argument");
    if ((a->prefix_len && !a->prefix) || (a->width && !a->table)) return set_error(IMI_E_ARG, "prefix_attn: no page list");
    if ((a->prefix_len || a->width) && (!a->k_pages || !a->v_pages || a->n_pages < 1))
        return set_error(IMI_E_ARG, "prefix_attn: no pages");
    if (a->width && a->table_stride < a->width) return set_error(IMI_E_ARG, "prefix_attn: table_stride below width");
    const int64_t row = (int64_t) a->n_head * a->head_dim;
    if (a->q_stride < row || a->out_stride < row || a->q_stride % 8 || a->out_stride % 8)
        return set_error(IMI_E_ARG, "prefix_attn: q and out rows are multiples of 8 elements apart, at least n_head * head_dim");
    if (!aligned(a->q, 16) || !aligned(a->k_pages, 16) || !aligned(a->v_pages, 16) || !aligned(a->out, 16) || !aligned(a->work, 16) ||
        !aligned(a->prefix, 4) || !aligned(a->table, 4) || !aligned(a->length, 4) || !aligned(a->lse, 4) || !aligned(a->status, 4))
        return set_error(IMI_E_ARG, "prefix_attn: a buffer is not aligned (q, pages, out and work: 16 bytes)");
    const PaPlan pl = pa_plan(a->rows, a->n_head, a->n_head_kv, a->head_dim, a->prefix_len, (long long) a->width * a->page);
    if (a->work_bytes < pl.bytes)
        return set_error(IMI_E_ARG, "prefix_attn: the workspace takes " + std::to_string(pl.bytes) + " bytes (imi_cuda_prefix_attn_work)");
    OnDevice on(device);
    if (!on.ok()) return set_error(IMI_E_NODEV, "no CUDA device " + std::to_string(device));
    if (!all_on_device({ a->q, a->k_pages, a->v_pages, a->prefix, a->table, a->length, a->out, a->lse, a->work, a->status }, device))
        return set_error(IMI_E_ARG, "prefix_attn: every buffer must be device memory of device " + std::to_string(device));
    PaArgs p = {};
    p.a = *a;
    p.shift = log2i(a->page);
    p.g = a->n_head / a->n_head_kv;
    p.sl2 = a->scale * LOG2E;
    p.pre_splits = pl.splits;
    p.pre_len = pl.len;
    p.mma = pl.mma;
    p.pair = pl.pair;
    p.tiles = pl.tiles;
    p.span = pl.span;
    p.per = pl.per;
    p.rtiles = pl.rtiles;
    p.off = (int *) a->work;
    const size_t slots = pl.pre_slots + pl.own_slots;
    p.pml = (float2 *) ((uint8_t *) a->work + pl.off_bytes);
    p.po = (float *) ((uint8_t *) a->work + pl.off_bytes + (slots * 8 + 255) / 256 * 256);
    p.own_slot0 = (int) pl.pre_slots;
    const bool half = a->type == IMI_F16;
    cudaError_t r = half ? raise_pa<__half>(device) : raise_pa<__nv_bfloat16>(device);
    if (r == cudaSuccess)
        r = half ? launch_pa_t<__half>(p, pl, (cudaStream_t) stream) : launch_pa_t<__nv_bfloat16>(p, pl, (cudaStream_t) stream);
    if (r != cudaSuccess) return set_error(IMI_E_CUDA, std::string("prefix_attn: ") + cudaGetErrorString(r));
    return IMI_OK;
}
