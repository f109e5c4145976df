// The shared prompt on the 5th-generation tensor cores (part of serve_attn.cu, inside its namespace): S = Q K^T and O += P V by
// tcgen05.mma with S, P and O in tensor memory, for many query rows on one list of positions.
//
// Rows are (conversation, head) pairs of one kv head, 128 to a tile; a CTA runs two streams of them against the same tiles of
// 128 positions (or, with at most 128 rows in all, one row tile against alternate position tiles), so that one stream's
// softmax overlaps the other's products. A thread of a softmax warp owns a row (a TMEM lane): no exchange between threads.
// P (two 16-bit values per column) is the product's A operand from TMEM; O stays in TMEM, and is rescaled only when a row's
// maximum has risen by more than 2^8 since the reference it was last scaled to (so a P is at most 2^8, which fp16 holds, and l
// is summed in 32 bits). At head_dim 64 S, P and O of both streams fill the 512 columns: QK(j+1) is issued as soon as S(j) is in
// the softmax's registers. At 128 P takes S's place, and QK(j+1) goes directly behind PV(j), which reads it (products of one
// thread run in the order of issue).
//   warp 0       K and V rows from their pages by tensor copies of up to 128 rows x 128 bytes into rings of tiles (128-byte
//                swizzle; the rows of a page that does not exist are read beyond the tensor's end, as zeros)
//   warp 1       zeroes V's rows that nobody sees, beyond the prompt's end in its last tile and below the lowest window in a unit's
//                first: what a page holds there may be anything
//   warp 3       issues the products
//   warps 4..7   softmax of stream 0, warps 8..11 of stream 1, with the registers that the others give up: a thread holds its
//                row's 128 scores
// K is [position][dimension], the B operand with K = dimension contiguous; V is the B operand with N = dimension contiguous.
// Bound by the exponentials: 16 per clock and SM, 2,048 clocks for two streams' tile; the products of head_dim 64 take half that.
// Measured: 1.64 us for two streams' tile (1.07 at that rate); 256 conversations of 32 heads on 16,384 positions 66 us in all.
#pragma once

constexpr int PM_M = 128, PM_N = 128, PM_ROWS = 2 * PM_M;
// query rows of a kv head up to which k_pa_pieces takes the prompt. A whole call by it and by k_pa_mma, on 2,000 positions: 8 rows
// 8.9 and 10.8 us, 16 9.1 and 10.8, 32 10.2 and 11.0, 64 11.6 and 11.8; on 16,000: 14.5 and 16.0, 17.6 and 16.9, 20.9 and 18.2, 28.9
// and 18.8
constexpr int PM_MIN_ROWS = 16;
constexpr int PM_MIN_TILES = 2;        // position tiles of a piece at least
constexpr int PM_BEGIN = 3;            // what a unit's beginning and end take, in tiles
constexpr int PM_MAX_TILES = 256;      // and at most (its page numbers are held in shared memory)
constexpr int PM_THREADS = 12 * 32;
// registers of a thread: at the launch (the host looks before the first one), then of the four warps that feed and the eight
// of the softmax; what those take has to be among the launch's, or they would wait for it for good
constexpr int PM_REGS = 168, PM_REGS_FEW = 80, PM_REGS_MANY = 208;
static_assert(4 * PM_REGS_FEW + 8 * PM_REGS_MANY <= 12 * PM_REGS, "setmaxnreg draws on the launch's own registers");
constexpr float PM_RISE = 8.0f;
constexpr int PM_HAND = 2;              // of four parts of a tile's exponentials, the one behind which the other stream begins
constexpr int PM_POLY = 4;              // every PM_POLY-th pair's exponentials by the FMA units

constexpr int PM_OROW = 80;            // bytes from row to row where a warp turns its part of O around: 16 values and padding

template <int D> struct PmSmem {
    static constexpr int TILE = PM_N * D * 2, NK = D == 64 ? 4 : 2, NV = D == 64 ? 4 : 2;
    static constexpr int Q = 0, K = Q + 2 * PM_M * D * 2, V = K + NK * TILE, IDS = V + NV * TILE,
                         OUT = IDS + PM_MAX_TILES * (PM_N / 16) * 4, BAR = OUT + 8 * 32 * PM_OROW, TOTAL = BAR + 512;
};

__device__ __forceinline__ void pm_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"((int) acc)
                 : "memory");
}
__device__ __forceinline__ void pm_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"((int) acc)
                 : "memory");
}
__device__ __forceinline__ void pm_commit(uint64_t *b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void pm_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
// true in one thread of the warp
__device__ __forceinline__ bool pm_elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void pm_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pm_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// a matrix descriptor with the 128-byte swizzle (layout 2 at bit 61, version 1 at bit 46); lbo and sbo in bytes
__device__ __forceinline__ uint64_t pm_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t) ((saddr >> 4) & 0x3FFF) | ((uint64_t) ((lbo >> 4) & 0x3FFF) << 16) | ((uint64_t) ((sbo >> 4) & 0x3FFF) << 32) |
           (1ull << 46) | (2ull << 61);
}
// kind::f16: D f32 (1 at bit 4), A and B both fp16 (0) or both bf16 (1) at bits 7 and 10, B with N contiguous: bit 16
template <typename T>
__device__ constexpr uint32_t pm_idesc(int m, int n, bool b_mn) {
    const uint32_t t = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (t << 7) | (t << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t) (n >> 3) << 17) | ((uint32_t) (m >> 4) << 24);
}
__device__ __forceinline__ void pm_ld32(uint32_t t, float (&v)[32]) {
    uint32_t *u = (uint32_t *) v;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
          "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
          "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(t));
}
__device__ __forceinline__ void pm_ld16(uint32_t t, float (&v)[16]) {
    uint32_t *u = (uint32_t *) v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
                   "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
                 : "r"(t));
}
__device__ __forceinline__ void pm_st32(uint32_t t, const float (&v)[32]) {
    const uint32_t *u = (const uint32_t *) v;
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
        "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
        "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]),
        "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]),
        "r"(u[31])
        : "memory");
}
__device__ __forceinline__ void pm_st16(uint32_t t, const uint32_t (&u)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(t),
                 "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
                 "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
                 : "memory");
}
__device__ __forceinline__ void pm_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 2^x for a pair by the FMA units: n the nearest integer, 2^(x - n) by the polynomial through its values at 6 Chebyshev nodes
// (relative error below 2^-21, ex2.approx's is 2^-22), times 2^n. Below 2^-126 0, as ex2.approx.ftz gives it (a masked score's
// weight, whatever V holds there), and a NaN stays one: hence the maximum that keeps it, and a product for 2^n where an addition
// to the exponent's bits would make numbers of both
__device__ __forceinline__ float pm_max_nan(float x, float y) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
    return m;
}
__device__ __forceinline__ float2 pm_exp2(float2 x) {
    x = make_float2(pm_max_nan(x.x, -127.0f), pm_max_nan(x.y, -127.0f));
    const float2 b = __fadd2_rn(x, make_float2(12582912.0f, 12582912.0f)),   // 1.5 * 2^23: n in the low bits
                 n = __fadd2_rn(b, make_float2(-12582912.0f, -12582912.0f)), f = __ffma2_rn(n, make_float2(-1.0f, -1.0f), x);
    float2 e = __ffma2_rn(f, make_float2(0.0013390863f, 0.0013390863f), make_float2(0.009676032f, 0.009676032f));
    e = __ffma2_rn(f, e, make_float2(0.05550357f, 0.05550357f));
    e = __ffma2_rn(f, e, make_float2(0.24022107f, 0.24022107f));
    e = __ffma2_rn(f, e, make_float2(0.6931472f, 0.6931472f));
    e = __ffma2_rn(f, e, make_float2(1.0f, 1.0f));
    return __fmul2_rn(e, make_float2(__int_as_float((__float_as_int(b.x) << 23) + 0x3f800000),    // n = -127: 0
                                     __int_as_float((__float_as_int(b.y) << 23) + 0x3f800000)));
}

template <typename T, int D>
__global__ void __launch_bounds__(PM_THREADS, 1) k_pa_mma(const __grid_constant__ PaArgs p, const __grid_constant__ CUtensorMap k_map,
                                                          const __grid_constant__ CUtensorMap v_map) {
    extern __shared__ __align__(1024) uint8_t sm_raw[];
    using L = PmSmem<D>;
    constexpr int NK = L::NK, NV = L::NV, CH = D / 8;
    constexpr bool APART = D == 64;                            // P beside S, not over it
    constexpr uint32_t TM_S = 0, TM_P = APART ? 2 * PM_N : 0, TM_O = APART ? 3 * PM_N : 2 * PM_N;   // TMEM columns, both streams'
    constexpr uint32_t P_STEP = APART ? PM_N / 2 : PM_N;       // from stream 0's P to stream 1's
    const imi_cuda_prefix_attn_args &a = p.a;
    uint8_t *sm = sm_raw + ((1024 - (smem_u32(sm_raw) & 1023)) & 1023);
    int *ids = (int *) (sm + L::IDS);
    uint64_t *k_full = (uint64_t *) (sm + L::BAR), *k_free = k_full + NK, *v_full = k_free + NK, *v_free = v_full + NV,
             *s_full = v_free + NV, *s_read = s_full + 2, *p_full = s_read + 2, *o_full = p_full + 2, *v_raw = o_full + 2, *q_full = v_raw + 2, *fin = q_full + 1,
             *turn_of = fin + 1;                               // [stream][warp]: the warp may begin its exponentials
    __shared__ uint32_t tmem_at;
    __shared__ int stop;
    __shared__ int low_of;                                     // the lowest position that a row of the unit sees
    // what a warp's threads agree on goes through a shuffle, so that the compiler keeps it, and the products' operands made of
    // it, in uniform registers: moved there for every product, issuing them took 2.5 us of a tile instead of 1
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(~0u, tid >> 5, 0);
    if (tid == 0) {
        for (int i = 0; i < NK; i++) { mbar_init(&k_full[i], 1); mbar_init(&k_free[i], 1); }
        for (int i = 0; i < NV; i++) { mbar_init(&v_full[i], 1); mbar_init(&v_free[i], 1); }
        for (int i = 0; i < 2; i++) { mbar_init(&s_full[i], 1); mbar_init(&s_read[i], 128); mbar_init(&p_full[i], 128); mbar_init(&o_full[i], 1); }
        for (int i = 0; i < 8; i++) mbar_init(&turn_of[i], 1);
        mbar_init(&v_raw[0], 1);
        mbar_init(&v_raw[1], 1);
        mbar_init(q_full, 256);
        mbar_init(fin, 1);
        stop = 0;
        fence_barrier_init();
    }
    if (warp == 3) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pm_fence_before();
    __syncthreads();
    pm_fence_after();
    const uint32_t tmem = __shfl_sync(~0u, tmem_at, 0);
    pdl_wait();
    pdl_trigger();

    auto wait = [&](uint64_t *b, uint32_t parity) -> bool {    // bounded: about a second, then the CTA gives up
        if (mbar_try_wait(b, parity)) return true;
        if (*(volatile int *) &stop) return false;
        if (mbar_wait(b, parity)) return true;
        stop = 1;
        if (a.status) atomicMax(a.status, IMI_DEV_WAIT);
        return false;
    };
    const int qrows = a.rows * p.g;
    // a negative scale turns q around; a scale of 0, which must not meet a mask's -infinity, is multiplied into it
    const float sl2 = p.sl2 == 0.0f ? 1.0f : fabsf(p.sl2);
    const bool turn = p.sl2 < 0.0f, flat = p.sl2 == 0.0f;
    const int line = p.rtiles * a.n_head_kv * p.span, end = min(line, ((int) blockIdx.x + 1) * p.per);
    int at = (int) blockIdx.x * p.per;
    struct Unit {
        int kvh, row0, piece, page0, t0, t1, n0, n1;           // position tiles [t0, t1), of them the streams'
        int low;                                               // the lowest position that a row of the unit sees
    };
    // the next unit's part, after the CTA is done with the one before: false where there is none. The page numbers are there
    // for warps 0..3 when it returns; the queries when q_full says so (the copies need not wait for them)
    int fr = -1, lo = 0;                                       // softmax: the thread's row, and what it sees from
    auto next = [&](Unit &w) -> bool {
        if (__syncthreads_or(at >= end || *(volatile int *) &stop)) return false;
        const int unit = at / p.span;
        w.piece = (int) blockIdx.x - unit * p.span / p.per;
        w.t0 = at - unit * p.span;
        w.t1 = min(p.tiles, w.t0 + (end - at));
        at += min(p.span - w.t0, end - at);
        w.kvh = unit / p.rtiles;
        w.row0 = (unit % p.rtiles) * (p.pair ? PM_M : PM_ROWS);
        w.page0 = (w.t0 * PM_N) >> p.shift;
        if (warp < 4) {                                        // the pages of this part, -1 for one that does not exist
            const int n = ((min(a.prefix_len, w.t1 * PM_N) - 1) >> p.shift) - w.page0 + 1;
            for (int i = tid; i < n; i += 128) {
                int id = __ldg(a.prefix + w.page0 + i);
                if ((unsigned) id >= (unsigned) a.n_pages) {
                    id = -1;
                    if (a.status) atomicMax(a.status, IMI_DEV_PAGE);
                }
                ids[i] = id;
            }
        } else {                                               // the queries
            const int x = tid - 128;
            fr = w.row0 + (p.pair ? x % PM_M : x);
            if (fr >= qrows) fr = -1;
            if (!p.pair || x < PM_M) {
                uint8_t *dst = sm + L::Q + (x / PM_M) * (PM_M * D * 2);
                const int r = x % PM_M;
                const T *q = fr >= 0 ? (const T *) a.q + fr / p.g * a.q_stride + ((long long) w.kvh * p.g + fr % p.g) * D : nullptr;
                uint4 v[CH];
#pragma unroll
                for (int c = 0; c < CH; c++) v[c] = q ? ldg16(q + 8 * c) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    if (turn) { v[c].x ^= 0x80008000u; v[c].y ^= 0x80008000u; v[c].z ^= 0x80008000u; v[c].w ^= 0x80008000u; }
                    if (flat)
#pragma unroll
                        for (int e = 0; e < 4; e++) (&v[c].x)[e] = Half2<T>::times_zero((&v[c].x)[e]);
                    *(uint4 *) (dst + (c / 8) * (PM_M * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[c];
                }
            }
            fence_proxy_async();
            pm_arrive(q_full);
        }
        if (a.window > 0) {                                    // what the rows see: tiles that none does are left out
            if (tid == 0) low_of = INT32_MAX;
            __syncthreads();
            if (warp >= 4) {
                const Seen v = fr >= 0 ? seen_of(p, fr / p.g) : Seen{ -1, 0, 0 };
                lo = v.len < 0 ? 0 : v.plo;                    // a row not in use, whose piece nobody reads, masks no tile
                const int least = __reduce_min_sync(~0u, v.len < 0 ? INT32_MAX : lo);
                if (lane == 0) atomicMin(&low_of, least);
            }
            __syncthreads();
            w.low = __shfl_sync(~0u, low_of, 0);
            w.t0 = max(w.t0, min(w.t1, w.low / PM_N));
        } else if (warp < 4) {
            asm volatile("bar.sync 1, 128;" ::: "memory");     // the page numbers
        }
        const int tiles = w.t1 - w.t0;
        w.n0 = p.pair ? (tiles + 1) / 2 : tiles;
        w.n1 = p.pair ? tiles / 2 : tiles;
        return true;
    };
    Unit w = {};
    // tiles of which nobody sees all V rows go past warp 1: the prompt's last by v_raw[1], a unit's first by v_raw[0]. At most one
    // of each in a part, so neither barrier is ever two phases ahead of its waiter
    auto at_end = [&](int t) { return (t + 1) * PM_N > a.prefix_len; };
    auto at_low = [&](int t) { return t * PM_N < w.low && !at_end(t); };
    // the page of a position (a multiple of 16, or in its group of 16) of the part
    auto id_at = [&](int pos) { return ids[(pos >> p.shift) - w.page0]; };

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PM_REGS_FEW));
        if (warp == 0) {
            // ---------------- copies ----------------
            const int box = min(a.page, PM_N), boxes = PM_N / box, none = a.n_pages * a.n_head_kv * a.page;
            int nk = 0, nv = 0;                                // tiles gone through the rings
            auto load = [&](const CUtensorMap &map, int tile, uint8_t *dst, uint64_t *full) {
                if (lane == 0) mbar_expect_tx(full, (uint32_t) L::TILE);
                __syncwarp();
                if (lane < boxes * (D / 64)) {                 // a box each: its rows, and which 64 dimensions
                    const int b = lane % boxes, half = lane / boxes, pos = tile * PM_N + b * box;
                    const int id = pos < a.prefix_len ? id_at(pos) : -1;
                    const int y = id >= 0 ? (id * a.n_head_kv + w.kvh) * a.page + (pos & (a.page - 1)) : none;
                    tma_load_2d(dst + half * (PM_N * 128) + b * box * 128, &map, 64 * half, y, full);
                }
                __syncwarp();
            };
            while (next(w)) {
                bool ok = true;
                for (int t = w.t0; t < w.t1 && ok; t++) {
                    const int ks = nk % NK, vs = nv % NV;
                    ok = __all_sync(~0u, wait(&k_free[ks], ((nk / NK) & 1) ^ 1));
                    if (!ok) break;
                    load(k_map, t, sm + L::K + ks * L::TILE, &k_full[ks]);
                    nk++;
                    ok = __all_sync(~0u, wait(&v_free[vs], ((nv / NV) & 1) ^ 1));
                    if (!ok) break;
                    load(v_map, t, sm + L::V + vs * L::TILE, at_end(t) ? &v_raw[1] : at_low(t) ? &v_raw[0] : &v_full[vs]);
                    nv++;
                }
                if (!ok) {                                     // copies in flight land before the memory goes (bounded)
                    for (int i = 0; i < NK && i < nk; i++) mbar_wait(&k_full[(nk - 1 - i) % NK], ((nk - 1 - i) / NK) & 1);
                    for (int i = 0; i < NV && i < nv; i++) mbar_wait(&v_full[(nv - 1 - i) % NV], ((nv - 1 - i) / NV) & 1);
                }
            }
        } else if (warp == 1) {
            // ---------------- V rows that nobody sees ----------------
            int nv = 0, nr[2] = { 0, 0 };
            while (next(w)) {
                auto clear = [&](int t, int end) {             // tile t: its rows below w.low, and from the prompt's end on
                    const int vs = (nv + t - w.t0) % NV, lo = min(PM_N, max(0, w.low - t * PM_N)), hi = min(PM_N, a.prefix_len - t * PM_N);
                    if (__all_sync(~0u, wait(&v_raw[end], nr[end] & 1))) {
                        uint8_t *v = sm + L::V + vs * L::TILE;
                        for (int half = 0; half < D / 64; half++)
                            for (int x = lane; x < PM_N * 8; x += 32)
                                if (x < lo * 8 || x >= hi * 8) *(uint4 *) (v + half * (PM_N * 128) + x * 16) = make_uint4(0, 0, 0, 0);
                        fence_proxy_async();
                        __syncwarp();
                        if (lane == 0) pm_arrive(&v_full[vs]);
                    }
                    nr[end]++;
                };
                if (w.t1 > w.t0 && at_low(w.t0)) clear(w.t0, 0);
                if (w.t1 > w.t0 && at_end(w.t1 - 1)) clear(w.t1 - 1, 1);
                nv += w.t1 - w.t0;
            }
        } else if (warp == 2) {
            while (next(w)) {}
        } else if (warp == 3) {
            // ---------------- products ----------------
            int units = 0, pn[2] = { 0, 0 }, rn[2] = { 0, 0 }, kn = 0, vn = 0;   // P and S tiles of the streams, tiles of the rings
            const uint32_t qk = pm_idesc<T>(PM_M, PM_N, false), pv = pm_idesc<T>(PM_M, D, true);
            // descriptors of the first tiles; the others' differ in the address alone (16-byte units, in the low bits)
            const uint64_t qd = pm_desc(smem_u32(sm + L::Q), 16, 1024), kd = pm_desc(smem_u32(sm + L::K), 16, 1024),
                           vd = pm_desc(smem_u32(sm + L::V), PM_N * 128, 1024);
            while (next(w)) {
                const int n0 = w.n0, n1 = w.n1;
                bool ok = __all_sync(~0u, wait(q_full, units++ & 1));
                auto issue_qk = [&](int st, int j) {
                    const int n = kn + (p.pair ? 2 * j + st : j), ks = n % NK;
                    ok = ok && __all_sync(~0u, wait(&k_full[ks], (n / NK) & 1));
                    if (!ok) return;
                    pm_fence_after();
                    if (pm_elect()) {
                        const uint64_t q = qd + (p.pair ? 0 : st) * (PM_M * D * 2 >> 4), k = kd + ks * (L::TILE >> 4);
#pragma unroll
                        for (int x = 0; x < D / 16; x++) {
                            const uint32_t o = ((x / 4) * (PM_N * 128) + (x % 4) * 32) >> 4;
                            pm_mma_ss(tmem + TM_S + st * PM_N, q + o, k + o, qk, x > 0);
                        }
                        pm_commit(&s_full[st]);
                        if (p.pair || st == 1) pm_commit(&k_free[ks]);
                    }
                    __syncwarp();
                };
                auto issue_pv = [&](int st, int j, bool last) {
                    const int n = vn + (p.pair ? 2 * j + st : j), vs = n % NV;
                    ok = ok && __all_sync(~0u, wait(&v_full[vs], (n / NV) & 1));
                    ok = ok && __all_sync(~0u, wait(&p_full[st], (pn[st] & 1)));
                    pn[st]++;
                    if (!ok) return;
                    pm_fence_after();
                    if (pm_elect()) {
                        const uint64_t v = vd + vs * (L::TILE >> 4);
#pragma unroll
                        for (int x = 0; x < PM_N / 16; x++)
                            pm_mma_ts(tmem + TM_O + st * D, tmem + TM_P + st * P_STEP + 8 * x, v + x * (2048 >> 4), pv, j > 0 || x > 0);
                        if (p.pair || st == 1) pm_commit(&v_free[vs]);
                        if (APART || last) pm_commit(&o_full[st]);
                    }
                    __syncwarp();
                };
                auto read = [&](int st) {                          // S is in the softmax's registers
                    ok = ok && __all_sync(~0u, wait(&s_read[st], rn[st] & 1));
                    rn[st]++;
                };
                if (n0 > 0 && ok) issue_qk(0, 0);
                if (n1 > 0 && ok) issue_qk(1, 0);
                for (int j = 0; j < n0 && ok; j++) {
                    if (APART) {
                        read(0);
                        if (j + 1 < n0) issue_qk(0, j + 1);
                        if (j < n1) read(1);
                        if (j + 1 < n1) issue_qk(1, j + 1);
                    }
                    issue_pv(0, j, j == n0 - 1);
                    if (!APART && j + 1 < n0) issue_qk(0, j + 1);
                    if (j < n1) issue_pv(1, j, j == n1 - 1);
                    if (!APART && j + 1 < n1) issue_qk(1, j + 1);
                }
                kn += w.t1 - w.t0;
                vn += w.t1 - w.t0;
            }
        }
    } else {
        // ---------------- softmax ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PM_REGS_MANY));
        const int st = (warp - 4) / 4;
        const uint32_t lanes = (uint32_t) ((warp & 3) * 32) << 16, S = tmem + TM_S + st * PM_N + lanes,
                       P = tmem + TM_P + st * P_STEP + lanes, O = tmem + TM_O + st * D + lanes;
        // The two warps of a scheduler, one of each stream, begin their exponentials in turn: in step, both would wait for the
        // same unit and then both for their products. With a quarter of them on the FMA units, 1.77 us of two streams' tile went to
        // 1.53 at head_dim 64; at 128, which waits for its products (P over S), neither made a difference, and both are left out
        uint64_t *my_turn = &turn_of[4 * st + (warp & 3)], *their_turn = &turn_of[4 * (1 - st) + (warp & 3)];
        int ns = 0, no = 0, nt = 0;                            // S tiles, O's commits, and turns, of this stream
        while (next(w)) {
            const int n = st ? w.n1 : w.n0;
            float m = -INFINITY, l = 0.0f;
            bool ok = true;
            for (int j = 0; j < n; j++, ns++) {
                const int pos = (w.t0 + (p.pair ? 2 * j + st : j)) * PM_N;
                ok = __all_sync(~0u, wait(&s_full[st], ns & 1));
                if (!ok) break;
                pm_fence_after();
                // which of the tile's positions this row sees: from `from` to `to`, but for groups of 16 without a page
                const int from = lo - pos, to = a.prefix_len - pos;
                unsigned groups = 0;
                if (lane < 8 && 16 * lane < to) groups = id_at(pos + 16 * lane) < 0;
                groups = __ballot_sync(~0u, groups);
                const bool masked = __any_sync(~0u, from > 0) || to < PM_N || groups;
                float v[PM_N];
#pragma unroll
                for (int c = 0; c < 4; c++) pm_ld32(S + 32 * c, *(float (*)[32]) (v + 32 * c));
                pm_wait_ld();
                if (APART) {
                    pm_fence_before();
                    pm_arrive(&s_read[st]);
                }
                if (masked)
#pragma unroll
                    for (int x = 0; x < PM_N; x++)
                        if (x < from || x >= to || (groups >> (x / 16) & 1)) v[x] = -INFINITY;
                float t4[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
                for (int x = 0; x < PM_N; x += 8)
#pragma unroll
                    for (int e = 0; e < 4; e++) t4[e] = fmaxf(t4[e], fmaxf(v[x + e], v[x + e + 4]));
                float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
                top = top == -INFINITY ? top : top * sl2;
                const bool raise = top > m + PM_RISE || (m == -INFINITY && top > m);
                const bool any = __any_sync(~0u, raise);
                // the product of the tile before reads P and adds to O: done before either is written
                if (APART && j > 0) {
                    ok = __all_sync(~0u, wait(&o_full[st], no & 1));
                    no++;
                    if (!ok) break;
                    pm_fence_after();
                }
                if (any) {
                    const float f = raise ? ex2(m - top) : 1.0f;   // m -infinity: 0
                    l *= f;
                    if (raise) m = top;
                    if (j > 0) {
                        float o[32];
#pragma unroll 1
                        for (int c = 0; c < D / 32; c++) {
                            pm_ld32(O + 32 * c, o);
                            pm_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] *= f;
                            pm_st32(O + 32 * c, o);
                        }
                    }
                }
                if (APART && (st == 1 || j > 0)) {
                    ok = __all_sync(~0u, wait(my_turn, nt & 1));
                    nt++;
                    if (!ok) break;
                }
                const float u = m == -INFINITY ? 0.0f : -m;
                const float2 s2 = make_float2(sl2, sl2), u2 = make_float2(u, u);
                float2 sum[2] = { make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f) };
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float2 x = __ffma2_rn(make_float2(v[32 * c + 2 * e], v[32 * c + 2 * e + 1]), s2, u2);
                        const float2 y = APART && e % PM_POLY == PM_POLY - 1 ? pm_exp2(x) : make_float2(ex2(x.x), ex2(x.y));
                        sum[e & 1] = __fadd2_rn(sum[e & 1], y);
                        pk[e] = Half2<T>::pack(y.x, y.y);
                    }
                    pm_st16(P + 16 * c, pk);
                    if (APART && c == PM_HAND && lane == 0 && (st == 0 ? j < w.n1 : j + 1 < w.n0)) pm_arrive(their_turn);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                pm_wait_st();
                pm_fence_before();
                pm_arrive(&p_full[st]);
            }
            // this row's piece
            const int i = fr / p.g, h = w.kvh * p.g + fr % p.g;
            const long long slot = ((long long) i * a.n_head + h) * p.pre_splits + (p.pair ? 2 * w.piece + st : w.piece);
            if (n > 0 && ok) {
                ok = __all_sync(~0u, wait(&o_full[st], no & 1));
                pm_fence_after();
            }
            if (fr >= 0) p.pml[slot] = make_float2(m, l);
            // O by 16 dimensions through shared memory, so that four threads write a row's 64 bytes: a row per thread, every store
            // would touch 32 lines (2.1 us of a piece against 0.5). Not unrolled: run once per piece, it waits for its instructions
            uint8_t *out = sm + L::OUT + (warp - 4) * 32 * PM_OROW;
            const long long to_row = fr >= 0 ? slot * D : -1;
            const bool real = n > 0 && ok;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
                float o[16];
                pm_ld16(O + c, o);
                pm_wait_ld();
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *(float4 *) (out + lane * PM_OROW + 4 * e) =
                        real ? make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int r = 8 * e + lane / 4;
                    const long long at_row = __shfl_sync(~0u, to_row, r);
                    if (at_row >= 0)
                        *(float4 *) (p.po + at_row + c + 4 * (lane % 4)) = *(const float4 *) (out + r * PM_OROW + 16 * (lane % 4));
                }
            }
            pm_fence_before();
            if (n > 0) no++;
        }
    }
    // products in flight end before their memory goes (bounded); copies have landed
    __syncthreads();
    if (warp == 3) {
        if (lane == 0) {
            pm_commit(fin);
            mbar_wait(fin, 0);
        }
        __syncwarp();
        pm_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}
