// serve_host.cuh — what the host sides of the operators over many sequences (serve.cu, serve16.cu) share: checks, the call's device, launches, the word of waits that ran out.
#pragma once
#include "serve.hpp"
#include "serve_cache.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <stdexcept>
#include <string>

namespace b200 {
namespace srv {

constexpr int MAX_SEQ = 4096;
constexpr int MAX_DEVICES = 64;

inline void need(bool ok, const std::string & what) { if (!ok) throw std::runtime_error(what); }
inline void cu(cudaError_t e, const char * what) {
    if (e == cudaSuccess) return;
    cudaGetLastError();                  // (it is this call's: who asks next, the other operators of this library among them, does not find it)
    throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

// the call's device while it runs, the caller's again behind it
struct On {
    int was = -1, device;
    int sms = 0;
    explicit On(int d) : device(d) {
        static std::atomic<int> known[MAX_DEVICES];            // SMs of the devices seen so far
        if (d < 0 || d >= MAX_DEVICES || !(sms = known[d].load())) {
            int n = 0;
            if (cudaGetDeviceCount(&n) != cudaSuccess) { cudaGetLastError(); n = 0; }
            need(n > 0, "no CUDA device visible: booster_b200 has no CPU fallback (the CUDA path is the product)");
            need(d >= 0 && d < n && d < MAX_DEVICES, "no such device: " + std::to_string(d));
            cu(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, d), "cudaDeviceGetAttribute");
            known[d].store(sms);
        }
        cu(cudaGetDevice(&was), "cudaGetDevice");
        if (was != d) cu(cudaSetDevice(d), "cudaSetDevice");
    }
    ~On() { if (was >= 0 && was != device) cudaSetDevice(was); }
};

// A word per device that a kernel raises when a bounded wait ran out, in pinned memory, so that the host reads it without waiting. Every call looks at it
inline std::atomic<int *> wait_words[MAX_DEVICES];
inline std::atomic<int> drill_polls;                                            // b200_kv4_drill
inline int * wait_word(int device) {
    static std::mutex lock;
    if (int * w = wait_words[device].load()) return w;
    std::lock_guard<std::mutex> hold(lock);
    if (int * w = wait_words[device].load()) return w;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;             // (this may be the first call inside a capture)
    cu(cudaThreadExchangeStreamCaptureMode(&mode), "cudaThreadExchangeStreamCaptureMode");
    void * p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, 64, cudaHostAllocPortable | cudaHostAllocMapped);
    cudaThreadExchangeStreamCaptureMode(&mode);
    cu(e, "cudaHostAlloc");
    *static_cast<volatile int *>(p) = 0;
    wait_words[device].store(static_cast<int *>(p));
    return static_cast<int *>(p);
}
inline void heed_waits(int device) {
    int * w = wait_words[device].load();
    if (w && *static_cast<volatile int *>(w) && __atomic_exchange_n(w, 0, __ATOMIC_ACQ_REL))
        throw std::runtime_error("a wait inside an earlier kv4_attention or kv16_attention on this device ran out: its results are worthless. This call has done nothing");
}

inline bool aligned(const void * p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline int log2_of(int x) { int l = 0; while ((1 << l) < x) l++; return l; }
inline int size_of(int dtype) { return dtype == B200_DTYPE_F32 ? 4 : 2; }

template <typename... P, typename... A>
void launch(void (*k)(P...), dim3 grid, int threads, size_t smem, void * stream, bool behind, int cluster, A &&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = (cudaStream_t) stream;
    cudaLaunchAttribute at[2];
    unsigned n = 0;
    if (behind) { at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization; at[n].val.programmaticStreamSerializationAllowed = 1; n++; }
    if (cluster > 1) { at[n].id = cudaLaunchAttributeClusterDimension; at[n].val.clusterDim.x = cluster; at[n].val.clusterDim.y = 1; at[n].val.clusterDim.z = 1; n++; }
    cfg.attrs = at; cfg.numAttrs = n;
    cu(cudaLaunchKernelEx(&cfg, k, static_cast<P>(args)...), "launch");
}

// leave for all the dynamic shared memory that a kernel can have beside what it holds statically, asked for once on each device. Calls of different sizes may come from several host threads:
// the limit does not depend on the call, so threads that set it together set the same
typedef std::atomic<bool> Limits[MAX_DEVICES];
template <typename K> void allow_smem(K * k, int device, Limits & set) {
    if (set[device].load()) return;
    cudaFuncAttributes at;
    int most = 0;
    cu(cudaFuncGetAttributes(&at, k), "cudaFuncGetAttributes");
    cu(cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, device), "cudaDeviceGetAttribute");
    cu(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int) at.sharedSizeBytes), "cudaFuncSetAttribute");
    set[device].store(true);
}

// tile_bytes: of 16 tokens of a KV head
inline Cache checked_cache(const b200_kv4 & c, const char * name, int tile_bytes) {
    const auto must = [&](bool ok, const char * what, int64_t got = INT64_MIN) {      // (the text is made where it is wanted: a call takes the host a few us)
        if (!ok) throw std::runtime_error(std::string(name) + ": " + what + (got == INT64_MIN ? "" : " (got " + std::to_string(got) + ")"));
    };
    must(c.head_dim == 64 || c.head_dim == 128, "head_dim is 64 or 128", c.head_dim);
    must(c.page_tokens >= 16 && c.page_tokens <= 1024 && (c.page_tokens & (c.page_tokens - 1)) == 0, "page_tokens is a power of two from 16 to 1024", c.page_tokens);
    must(c.n_head_kv >= 1 && c.n_head_kv <= 1024, "n_head_kv from 1 to 1024");
    must(c.n_pages >= 1, "a pool of one page at least");
    must(c.n_slots >= 1 && c.max_pages >= 1 && (int64_t) c.max_pages * c.page_tokens <= (1 << 30), "a table of one slot and one page at least, of 2^30 tokens a slot at most");
    static_assert(MAX_SEQ == 4096, "the text");
    must(c.n_seq >= 0 && c.n_seq <= MAX_SEQ, "from 0 to 4096 sequences a step", c.n_seq);
    must(c.n_rows >= 0 && c.n_rows <= (1 << 24), "from 0 to 2^24 rows a step", c.n_rows);
    must(c.page_stride >= (int64_t) c.n_head_kv * c.page_tokens / 16 * tile_bytes && c.page_stride % 16 == 0, "page_stride holds a page and is a multiple of 16 bytes", c.page_stride);
    must(c.table_stride >= c.max_pages, "table_stride is max_pages at least", c.table_stride);
    must(c.pool && c.table && c.held && c.first, "null pointer");
    must(aligned(c.pool, 16), "the pool starts on 16 bytes");
    must(aligned(c.table, 4) && aligned(c.held, 4) && aligned(c.first, 4) && aligned(c.slots, 4), "tables of int32 start on 4 bytes");
    return Cache{static_cast<uint8_t *>(c.pool), c.page_stride, c.n_pages, log2_of(c.page_tokens), c.n_head_kv, c.table, c.table_stride, c.n_slots, c.max_pages, c.held, c.slots, c.first, c.n_seq, c.n_rows};
}
inline void check_dtype(int dtype, bool f32) {
    need(dtype == B200_DTYPE_BF16 || dtype == B200_DTYPE_F16 || (f32 && dtype == B200_DTYPE_F32), f32 ? "dtype is B200_DTYPE_F32, _BF16 or _F16" : "dtype is B200_DTYPE_BF16 or _F16");
}

inline void check_work(const void * work, int64_t bytes, int64_t wanted) {
    need(work && aligned(work, 16), "the workspace starts on 16 bytes");
    need(bytes >= wanted, "the workspace has " + std::to_string(bytes) + " bytes, " + std::to_string(wanted) + " are needed");
}
}  // namespace srv
}  // namespace b200
