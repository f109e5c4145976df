// What the serving operators' files (serve_pages.cu, serve_attn.cu, serve_sample.cu) share on the host: the error
// message of the library, the checks of a call's device and buffers, and the launch with programmatic serialization.
#pragma once
#include "../../include/imi_cuda.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <mutex>
#include <string>

namespace imi {
struct SessDev;   // common.cuh: a conversation's scalars on the device

imi_cuda_status set_error(imi_cuda_status st, const std::string &msg);   // engine.cpp: the text of imi_cuda_error()

// How sampling cuts n rows of vocab words: `ctas` per row (a cluster), `share` words for each of them but the last, held in SM_NW
// parts of `seg` (a multiple of SM_TILE). CTAs per row: as many as hold the row, more while the call has few (SM_FEW) and a CTA
// keeps a tile per warp. More CTAs help the passes over the row (one row of 97,496 by nucleus: 22 us with 8, 25.9 with 4; 16 of
// 32,000: 15.4 with 4, 38 with 1), and cost where the short way does (32 rows of 32,000 by top-k: 8.1 us with 4, 15.4 with 8; 64 of
// 8,000: 7.1 with 2, 8.9 with 4). The words are shared out evenly, by fours (the loads' width): CTAs filled to their last part one
// after the other leave some cluster's last ones with few words or none, whose threads' maxima then bound nothing, and the row
// misses its short list (one row of 50,257 by top-k 50: 23.9 us so, 7.4 shared out)
constexpr int SM_NW = 16;                // warps of a CTA
constexpr int SM_TILE = 128;             // words of a warp's load: four per lane
constexpr int SM_MAX_CLUSTER = 8;
constexpr int SM_SLICE = 32768;          // words a CTA holds at most
constexpr int SM_LIST = 768;             // words of a list at most
constexpr int SM_AIM(int c) { return c == 1 ? 600 : c == 2 ? 480 : 425; }   // words listed for top-p alone, about
constexpr int SM_FEW(int c) { return c < 4 ? 96 : 48; }   // CTAs of a call, of c per row, below which its rows get twice as many
// rank: for top-p alone, which of a CTA's threads' maxima bounds the list. Of L threads with q words each, a share f of the words is
// above the (1 - (1 - f)^q) L-th largest of their maxima; f is set for SM_AIM words of the row, L and q are the last CTA's. The more
// CTAs, the more their lowest bound lists beside that: about 500 words with 2 to 8; one CTA leaves 4 standard deviations to SM_LIST.
// (A fixed rank of 384 over the CTAs asked one CTA for more maxima than it had, or for so low a one that the list overflowed: 100
// rows of 5,000 by nucleus 0.9 22.1 us so, 14.8 by this.) A row that fits the list whole is listed whole: a rank beyond all threads
struct SampleSplit {
    int ctas, seg, share, rank;
};
inline SampleSplit sample_split(int n, int vocab) {
    int c = 1;
    while (c < SM_MAX_CLUSTER && ((vocab + c - 1) / c > SM_SLICE || (n * c < SM_FEW(c) && vocab > c * SM_NW * SM_TILE))) c *= 2;
    const int share = ((vocab + c - 1) / c + 3) / 4 * 4;
    const int seg = ((share + SM_NW - 1) / SM_NW + SM_TILE - 1) / SM_TILE * SM_TILE, last = vocab - (c - 1) * share;
    const int lanes = last / seg * 32 + std::min(32, (last % seg + 3) / 4);
    const double above = 1.0 - std::pow(1.0 - std::min(1.0, (double) SM_AIM(c) / vocab), (double) last / lanes);
    return { c, seg, share, vocab <= SM_LIST ? 32 * SM_NW : std::max(1, (int) (above * lanes)) };
}

// serve_sample.cu: sampling of checked arguments with `device` current; rows (or null): device pointers of the rows' scores,
// states (or null): the conversations whose last pick, with its score, the words become
cudaError_t launch_sample(int device, const imi_cuda_sample_args &a, const void *const *rows, SessDev *const *states, cudaStream_t st);

// makes `device` current while it lives; ok() false: there is no such device
class OnDevice {
    int prev_ = -1;
    bool ok_ = false;

public:
    explicit OnDevice(int device) {
        if (device < 0 || cudaGetDevice(&prev_) != cudaSuccess) {
            cudaGetLastError();
            return;
        }
        ok_ = prev_ == device || cudaSetDevice(device) == cudaSuccess;
        if (!ok_) cudaGetLastError();
    }
    ~OnDevice() {
        int now = -1;
        if (prev_ >= 0 && cudaGetDevice(&now) == cudaSuccess && now != prev_) cudaSetDevice(prev_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;
    bool ok() const { return ok_; }
};

// every non-null pointer is device memory of `device` (or managed memory)
inline bool all_on_device(std::initializer_list<const void *> ps, int device) {
    for (const void *p : ps) {
        if (!p) continue;
        cudaPointerAttributes at = {};
        if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
            cudaGetLastError();
            return false;
        }
        if (!(at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == device))) return false;
    }
    return true;
}

inline bool aligned(const void *p, size_t n) { return ((uintptr_t) p) % n == 0; }
inline bool page_ok(int page) { return page >= 16 && page <= 256 && (page & (page - 1)) == 0; }
inline int log2i(int x) {
    int k = 0;
    while ((1 << k) < x) k++;
    return k;
}

// a launch that may start while its predecessor on the stream drains: the kernel calls pdl_wait() before it reads or
// writes anything the predecessor may touch
inline cudaError_t launch_pdl(const void *fn, dim3 grid, int threads, size_t smem, cudaStream_t st, void **args,
                              int cluster = 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelExC(&cfg, fn, args);
}

// raises a kernel's shared-memory limit once per device (the attribute belongs to the device that is current)
constexpr int MAX_DEVICES = 64;
struct SmemLimit {
    std::mutex mu;
    bool done[MAX_DEVICES] = {};
    cudaError_t raise(int device, std::initializer_list<const void *> fns, int bytes) {
        std::lock_guard<std::mutex> g(mu);
        if (device < MAX_DEVICES && done[device]) return cudaSuccess;
        for (const void *f : fns) {
            const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
            if (e != cudaSuccess) return e;
        }
        if (device < MAX_DEVICES) done[device] = true;
        return cudaSuccess;
    }
};
}  // namespace imi
