// serve.cu — host side of the operators of a server that runs many sequences at once (serve.hpp): checks of arguments, launch shapes, launches on the caller's stream.
#include "serve.hpp"
#include "serve_cache.cuh"
#include "serve_attn.cuh"
#include "serve_prompt.cuh"
#include "serve_pages.cuh"
#include "serve_sample.cuh"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <stdexcept>
#include <string>

namespace b200 {
namespace {

using namespace srv;

constexpr int MAX_DEVICES = 64;

void need(bool ok, const std::string & what) { if (!ok) throw std::runtime_error(what); }
void cu(cudaError_t e, const char * what) {
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

// A word per device that k_kv4_prompt raises when a bounded wait ran out, in pinned memory, so that the host reads it without waiting. Every call looks at it
std::atomic<int *> wait_words[MAX_DEVICES];
std::atomic<int> drill_polls;                                            // b200_kv4_drill
int * wait_word(int device) {
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
void heed_waits(int device) {
    int * w = wait_words[device].load();
    if (w && *static_cast<volatile int *>(w) && __atomic_exchange_n(w, 0, __ATOMIC_ACQ_REL))
        throw std::runtime_error("a wait inside an earlier kv4_attention on this device ran out: its results are worthless. This call has done nothing");
}

bool aligned(const void * p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int log2_of(int x) { int l = 0; while ((1 << l) < x) l++; return l; }
int size_of(int dtype) { return dtype == B200_DTYPE_F32 ? 4 : 2; }

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

Cache checked(const b200_kv4 & c) {
    need(c.head_dim == 64 || c.head_dim == 128, "kv4: head_dim is 64 or 128 (got " + std::to_string(c.head_dim) + ")");
    need(c.page_tokens >= 16 && c.page_tokens <= 1024 && (c.page_tokens & (c.page_tokens - 1)) == 0, "kv4: page_tokens is a power of two from 16 to 1024 (got " + std::to_string(c.page_tokens) + ")");
    need(c.n_head_kv >= 1 && c.n_head_kv <= 1024, "kv4: n_head_kv from 1 to 1024");
    need(c.n_pages >= 1, "kv4: a pool of one page at least");
    need(c.n_slots >= 1 && c.max_pages >= 1 && (int64_t) c.max_pages * c.page_tokens <= (1 << 30), "kv4: a table of one slot and one page at least, of 2^30 tokens a slot at most");
    need(c.n_seq >= 0 && c.n_seq <= AT_MAX_SEQ, "kv4: from 0 to " + std::to_string(AT_MAX_SEQ) + " sequences a step");
    need(c.n_rows >= 0 && c.n_rows <= (1 << 24), "kv4: from 0 to 2^24 rows a step");
    need(c.page_stride >= (int64_t) c.n_head_kv * c.page_tokens / 16 * 18 * c.head_dim && c.page_stride % 16 == 0, "kv4: page_stride holds a page and is a multiple of 16 bytes");
    need(c.table_stride >= c.max_pages, "kv4: table_stride is max_pages at least");
    need(c.pool && c.table && c.held && c.first, "kv4: null pointer");
    need(aligned(c.pool, 16), "kv4: the pool starts on 16 bytes");
    need(aligned(c.table, 4) && aligned(c.held, 4) && aligned(c.first, 4) && aligned(c.slots, 4), "kv4: tables of int32 start on 4 bytes");
    return Cache{static_cast<uint8_t *>(c.pool), c.page_stride, c.n_pages, log2_of(c.page_tokens), c.n_head_kv, c.table, c.table_stride, c.n_slots, c.max_pages, c.held, c.slots, c.first, c.n_seq, c.n_rows};
}
void check_dtype(int dtype, bool f32) {
    need(dtype == B200_DTYPE_BF16 || dtype == B200_DTYPE_F16 || (f32 && dtype == B200_DTYPE_F32), f32 ? "dtype is B200_DTYPE_F32, _BF16 or _F16" : "dtype is B200_DTYPE_BF16 or _F16");
}

// heads of a row one after the other in a warp only where there are rows enough to fill the card without. Rows of 8 heads written and read by one pass / by four, us: 48 6.2 / 8.9,
// 700 9.3 / 11.1, 2100 11.9 / 11.9, 8100 32 / 25
int row_passes(const b200_kv4 & c) { return (int64_t) c.n_rows * c.n_head_kv > 16384 ? 4 : 1; }
int row_parts(const b200_kv4 & c) { const int per = row_passes(c) * (128 / c.head_dim); return (c.n_head_kv + per - 1) / per; }
unsigned row_blocks(const b200_kv4 & c) { return (unsigned) (((int64_t) c.n_rows * row_parts(c) + 7) / 8); }
template <typename T> void append_as(const b200_kv4 & c, const Cache & d, const void * k, int64_t kr, int64_t kh, const void * v, int64_t vr, int64_t vh) {
    const RowSrc<T> src = {static_cast<const T *>(k), kr, kh, static_cast<const T *>(v), vr, vh, aligned(k, 4 * sizeof(T)) && aligned(v, 4 * sizeof(T)) && !((kr | kh | vr | vh) & 3)};
    const auto rows = [&](auto kernel) { launch(kernel, dim3(row_blocks(c)), 256, 0, c.stream, false, 1, d, src, row_parts(c)); };
    if (row_passes(c) == 1) c.head_dim == 128 ? rows(k_kv4_append<T, 128, 1>) : rows(k_kv4_append<T, 64, 1>);
    else c.head_dim == 128 ? rows(k_kv4_append<T, 128, 4>) : rows(k_kv4_append<T, 64, 4>);
}
template <typename T> void read_as(const b200_kv4 & c, const Cache & d, void * k, void * v) {
    T * ko = static_cast<T *>(k), * vo = static_cast<T *>(v);
    const auto rows = [&](auto kernel) { launch(kernel, dim3(row_blocks(c)), 256, 0, c.stream, false, 1, d, ko, vo, row_parts(c)); };
    if (row_passes(c) == 1) c.head_dim == 128 ? rows(k_kv4_read<T, 128, 1>) : rows(k_kv4_read<T, 64, 1>);
    else c.head_dim == 128 ? rows(k_kv4_read<T, 128, 4>) : rows(k_kv4_read<T, 64, 4>);
}

// attention of few rows: column tiles of 8, two side by side where one does not hold a sequence's columns (48 sequences of 3000, 4 columns: one 46 us, two 58; 12: 82 and 64)
int attend_nt(int group, int max_rows) { return (int64_t) group * max_rows <= 8 ? 1 : 2; }
size_t attend_before_bytes(int n_seq) { return ((size_t) (n_seq + 2) * 8 + 255) / 256 * 256; }
size_t attend_bytes(int n_seq, int head_dim, int nt, int sms) {
    const size_t slots = 2 * (size_t) sms * at_blocks(nt) * AT_WARPS, cols = 8 * (size_t) nt;
    return attend_before_bytes(n_seq) + slots * cols * (head_dim + 2) * 4;
}
template <int HD, int NT, typename T> void attend_as(const AttendArgs & a, int device, int sms, void * stream) {
    static Limits set;
    const size_t smem = at_ring_bytes(HD) + (size_t) (a.c.n_seq + 1) * 8;
    const auto kernel = k_kv4_attend<HD, NT, T>;
    allow_smem(kernel, device, set);
    launch(kernel, dim3(sms * at_blocks(NT)), AT_WARPS * 32, smem, stream, false, 1, a);
    const int64_t items = (int64_t) a.c.n_rows * a.c.n_kv * a.group;
    // parts a unit has on average, where every sequence has rows: few are one warp's to add, many sixteen's. One / four / sixteen warps, us, 8 KV heads: one sequence of 20 000 39 / 22 / 16,
    // 6 of 4000 20 / 17 / 17, 24 of 4000 33 / 32 / 38, 48 of 3000 43 / 45 / 54, 300 of 100 27 / 38 / 81
    const int64_t parts = (int64_t) sms * at_blocks(NT) * AT_WARPS / ((int64_t) a.c.n_seq * a.c.n_kv);
    if (parts > 32) launch(k_kv4_join<HD, NT, T, 16>, dim3((unsigned) items), 512, 0, stream, true, 1, a);
    else if (parts > 8) launch(k_kv4_join<HD, NT, T, 4>, dim3((unsigned) items), 128, 0, stream, true, 1, a);
    else launch(k_kv4_join<HD, NT, T, 1>, dim3((unsigned) ((items + 7) / 8)), 256, 0, stream, true, 1, a);
}
template <int HD, typename T> void attend_nt_as(const AttendArgs & a, int nt, int device, int sms, void * stream) {
    nt == 1 ? attend_as<HD, 1, T>(a, device, sms, stream) : attend_as<HD, 2, T>(a, device, sms, stream);
}

// attention of prompts' portions
int64_t prompt_entries(const b200_kv4 & c, int group) { return (int64_t) c.n_rows * group / PR_COLS + c.n_seq + 1; }
struct PromptWork { int64_t entries, first, ml, part, bytes; };       // places in the workspace; `before` is first
PromptWork prompt_work(const b200_kv4 & c, int group, int sms) {
    const auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t n = prompt_entries(c, group), slots = 2 * (int64_t) sms * PR_COLS;
    PromptWork w;
    w.entries = up((n + 2) * 8);
    w.first = w.entries + up(n * (int64_t) sizeof(Entry));
    w.ml = w.first + up((sms + 2) * 4);
    w.part = w.ml + up(slots * 8);
    w.bytes = w.part + slots * c.head_dim * 4;
    return w;
}
template <int HD, typename T> void prompt_as(const PromptArgs & p, int64_t entries, int device, int sms, void * stream) {
    static Limits set;
    const auto kernel = k_kv4_prompt<HD, T>;
    allow_smem(kernel, device, set);
    launch(k_kv4_prompt_plan, dim3(1), 1024, (size_t) (p.a.c.n_seq + 1) * 4, stream, false, 1, p, sms);
    launch(kernel, dim3(sms), PR_THREADS, PromptSmem<HD>::BYTES, stream, true, 1, p);
    launch(k_kv4_prompt_join<HD, T>, dim3((unsigned) (entries * (PR_COLS / 32)), (unsigned) p.a.c.n_kv), 256, 0, stream, true, 1, p);
}

Pages checked(const b200_pages & p, bool pool) {
    need(p.page_tokens >= 16 && p.page_tokens <= 1024 && (p.page_tokens & (p.page_tokens - 1)) == 0, "pages: page_tokens is a power of two from 16 to 1024 (got " + std::to_string(p.page_tokens) + ")");
    need(p.n_pages >= 1 && p.n_pages <= PG_MAX_PAGES, "pages: from 1 to 2^20 pages");
    need(p.n_slots >= 1 && p.n_slots <= PG_MAX_SLOTS, "pages: from 1 to 2^18 slots");
    need(p.max_pages >= 1 && (int64_t) p.max_pages * p.page_tokens <= (1 << 30), "pages: from one page to 2^30 tokens a slot");
    need(p.table_stride >= p.max_pages, "pages: table_stride is max_pages at least");
    need(p.table && p.held && p.refs, "pages: null pointer");
    need(aligned(p.table, 4) && aligned(p.held, 4) && aligned(p.refs, 4), "pages: tables of int32 start on 4 bytes");
    int64_t bytes = 0;
    if (pool) {
        need(p.head_dim == 64 || p.head_dim == 128, "pages: head_dim is 64 or 128 (got " + std::to_string(p.head_dim) + ")");
        need(p.n_head_kv >= 1 && p.n_head_kv <= 1024 && p.n_layer >= 1 && p.n_layer <= 65536, "pages: n_head_kv from 1 to 1024, n_layer from 1 to 65536");
        bytes = (int64_t) p.n_head_kv * p.page_tokens / 16 * 18 * p.head_dim;
        need(p.pool && aligned(p.pool, 16), "pages: the pool starts on 16 bytes");
        need(p.page_stride >= bytes && p.page_stride % 16 == 0 && p.layer_stride % 16 == 0 && (p.n_layer == 1 || p.layer_stride >= bytes), "pages: strides hold a page and are multiples of 16 bytes");
    }
    return Pages{p.table, p.table_stride, p.n_slots, p.max_pages, p.held, p.refs, p.n_pages, log2_of(p.page_tokens), static_cast<uint8_t *>(p.pool), p.layer_stride, p.page_stride,
                 p.n_layer, p.n_head_kv, 18 * p.head_dim};
}
size_t words_bytes(int n) { return (size_t) ((n + 31) / 32) * 4; }
void check_work(const void * work, int64_t bytes, int64_t wanted) {
    need(work && aligned(work, 16), "the workspace starts on 16 bytes");
    need(bytes >= wanted, "the workspace has " + std::to_string(bytes) + " bytes, " + std::to_string(wanted) + " are needed");
}
void move_pages(const b200_pages & p, const Pages & d, const int32_t * plan, int n, bool parts, const int32_t * moved_to, int sms) {
    launch(k_pages_move, dim3(sms * 4), 256, 0, p.stream, true, 1, d, plan, n, parts, moved_to);
}

template <typename T> void sample_as(const SampleArgs & a, int cluster, int device, void * stream) {
    static Limits set;
    const size_t smem = SA_FIXED + ((size_t) a.slice * sizeof(T) + 15) / 16 * 16;
    allow_smem(k_sample<T>, device, set);
    launch(k_sample<T>, dim3((unsigned) (a.n_rows * cluster)), SA_THREADS, smem, stream, false, cluster, a);
}

}  // namespace

void kv4_append(const b200_kv4 & c, int dtype, const void * k, int64_t k_row, int64_t k_head, const void * v, int64_t v_row, int64_t v_head) {
    const Cache d = checked(c);
    check_dtype(dtype, true);
    need(c.n_rows == 0 || (k && v && aligned(k, size_of(dtype)) && aligned(v, size_of(dtype))), "kv4_append: k and v are pointers to whole entries");
    On on(c.device);
    heed_waits(c.device);
    if (c.n_seq == 0 || c.n_rows == 0) return;
    if (dtype == B200_DTYPE_F32) append_as<float>(c, d, k, k_row, k_head, v, v_row, v_head);
    else if (dtype == B200_DTYPE_BF16) append_as<__nv_bfloat16>(c, d, k, k_row, k_head, v, v_row, v_head);
    else append_as<__half>(c, d, k, k_row, k_head, v, v_row, v_head);
}

void kv4_read(const b200_kv4 & c, int dtype, void * k, void * v) {
    const Cache d = checked(c);
    check_dtype(dtype, true);
    need(c.n_rows == 0 || (k && v && aligned(k, 16) && aligned(v, 16)), "kv4_read: k and v start on 16 bytes");
    On on(c.device);
    heed_waits(c.device);
    if (c.n_seq == 0 || c.n_rows == 0) return;
    if (dtype == B200_DTYPE_F32) read_as<float>(c, d, k, v);
    else if (dtype == B200_DTYPE_BF16) read_as<__nv_bfloat16>(c, d, k, v);
    else read_as<__half>(c, d, k, v);
}

static void check_heads(const b200_kv4 & c, int n_head, int max_rows) {
    need(n_head >= c.n_head_kv && n_head % std::max(1, c.n_head_kv) == 0 && (int64_t) c.n_rows * n_head <= (1 << 30), "kv4_attention: n_head is a multiple of n_head_kv (got " + std::to_string(n_head) + " and " + std::to_string(c.n_head_kv) + "), and rows x heads up to 2^30");
    need(max_rows >= 1 && max_rows <= (1 << 24), "kv4_attention: max_rows is the largest number of rows of a sequence");
}

// Columns of a sequence (rows x query heads of a KV head) from which its tiles are worth making fp16 for the tensor cores' larger products. Where sequences x KV heads give the SMs few units
// the finer pieces of the form for few rows pay longer. Few rows / many rows, us, 8 KV heads, group 4: one sequence of 8000 positions, 64 columns 25 / 38, 128 39 / 40, 256 64 / 44;
// 8 of 2000, 48 columns 27 / 31, 64 32 / 31, 96 40 / 32; 48 of 3000, 48 columns 120 / 143, 64 151 / 144, 96 215 / 144
bool is_prompt(const b200_kv4 & c, int group, int max_rows) { return (int64_t) group * max_rows > ((int64_t) c.n_seq * c.n_head_kv < 64 ? 128 : 48); }

int64_t kv4_attention_workspace(const b200_kv4 & c, int n_head, int max_rows) {
    checked(c);
    check_heads(c, n_head, max_rows);
    On on(c.device);
    if (is_prompt(c, n_head / c.n_head_kv, max_rows)) return prompt_work(c, n_head / c.n_head_kv, on.sms).bytes;
    return (int64_t) attend_bytes(c.n_seq, c.head_dim, attend_nt(n_head / c.n_head_kv, max_rows), on.sms);
}

void kv4_attention(const b200_kv4 & c, int dtype, const void * q, int64_t q_row, int64_t q_head, int n_head, float scale, int window, int max_rows, void * out, void * work, int64_t work_bytes) {
    AttendArgs a = {};
    a.c = checked(c);
    check_dtype(dtype, false);
    check_heads(c, n_head, max_rows);
    need(c.n_rows == 0 || (q && out && aligned(q, 2) && aligned(out, 16)), "kv4_attention: q points to whole entries, out starts on 16 bytes");
    need(std::isfinite(scale), "kv4_attention: scale is a finite number");
    need(window >= 0, "kv4_attention: window is a number of positions, or 0 for all");
    On on(c.device);
    heed_waits(c.device);
    if (c.n_seq == 0 || c.n_rows == 0) return;
    a.q = q; a.q_row = q_row; a.q_head = q_head; a.out = out;
    a.q_whole = aligned(q, 16) && !((q_row | q_head) & 7);
    a.group = n_head / c.n_head_kv;
    a.scale_log2 = scale * 1.44269504088896341f;
    a.window = window;
    uint8_t * w = static_cast<uint8_t *>(work);
    if (is_prompt(c, a.group, max_rows)) {
        const PromptWork at = prompt_work(c, a.group, on.sms);
        check_work(work, work_bytes, at.bytes);
        const int drill = drill_polls.load();
        PromptArgs p = {a, (int) prompt_entries(c, a.group), reinterpret_cast<Entry *>(w + at.entries), reinterpret_cast<int *>(w + at.first), wait_word(c.device),
                        drill ? (uint32_t) drill : PR_POLLS, drill ? 1 << 19 : 4};
        const int64_t n = prompt_entries(c, a.group);
        p.a.before = reinterpret_cast<long long *>(w);
        p.a.ml = reinterpret_cast<float *>(w + at.ml);
        p.a.part = reinterpret_cast<float *>(w + at.part);
        if (dtype == B200_DTYPE_BF16) c.head_dim == 128 ? prompt_as<128, __nv_bfloat16>(p, n, c.device, on.sms, c.stream) : prompt_as<64, __nv_bfloat16>(p, n, c.device, on.sms, c.stream);
        else c.head_dim == 128 ? prompt_as<128, __half>(p, n, c.device, on.sms, c.stream) : prompt_as<64, __half>(p, n, c.device, on.sms, c.stream);
        return;
    }
    const int nt = attend_nt(a.group, max_rows);
    check_work(work, work_bytes, (int64_t) attend_bytes(c.n_seq, c.head_dim, nt, on.sms));
    const size_t slots = 2 * (size_t) on.sms * at_blocks(nt) * AT_WARPS;
    a.before = reinterpret_cast<long long *>(w);
    a.ml = reinterpret_cast<float *>(w + attend_before_bytes(c.n_seq));
    a.part = a.ml + slots * 8 * nt * 2;
    if (dtype == B200_DTYPE_BF16) c.head_dim == 128 ? attend_nt_as<128, __nv_bfloat16>(a, nt, c.device, on.sms, c.stream) : attend_nt_as<64, __nv_bfloat16>(a, nt, c.device, on.sms, c.stream);
    else c.head_dim == 128 ? attend_nt_as<128, __half>(a, nt, c.device, on.sms, c.stream) : attend_nt_as<64, __half>(a, nt, c.device, on.sms, c.stream);
}

int64_t pages_workspace(const b200_pages & p, int n) {
    need(p.n_pages >= 1 && p.n_pages <= PG_MAX_PAGES && n >= 0 && n <= PG_MAX_PAGES, "pages_workspace: from 1 to 2^20 pages");
    return 4 * (int64_t) (PLAN_HEAD + 3 * (int64_t) std::max(n, 1));
}

void pages_reserve(const b200_pages & p, const int32_t * slots, const int32_t * first, int n, int32_t * status) {
    const Pages d = checked(p, false);
    need(n >= 0 && n <= PG_MAX_N, "pages_reserve: from 0 to " + std::to_string(PG_MAX_N) + " sequences");
    need(first && status, "pages_reserve: null pointer");
    need(slots || n <= p.n_slots, "pages_reserve: more sequences than slots");
    On on(p.device);
    heed_waits(p.device);
    static Limits set;
    const size_t smem = words_bytes(p.n_pages) + words_bytes(p.n_slots);
    allow_smem(k_pages_reserve, p.device, set);
    launch(k_pages_reserve, dim3(1), PG_THREADS, smem, p.stream, false, 1, d, slots, first, n, status);
}

void pages_fork(const b200_pages & p, const int32_t * parents, const int32_t * children, int n, int32_t * status, void * work, int64_t work_bytes) {
    const Pages d = checked(p, true);
    need(n >= 0 && n <= PG_MAX_N, "pages_fork: from 0 to " + std::to_string(PG_MAX_N) + " pairs");
    need(status && ((parents && children) || n == 0), "pages_fork: null pointer");
    check_work(work, work_bytes, pages_workspace(p, n));
    On on(p.device);
    heed_waits(p.device);
    static Limits set;
    const size_t smem = words_bytes(p.n_pages) + words_bytes(p.n_slots);
    allow_smem(k_pages_fork, p.device, set);
    int32_t * plan = static_cast<int32_t *>(work);
    launch(k_pages_fork, dim3(1), PG_THREADS, smem, p.stream, false, 1, d, parents, children, n, status, plan);
    move_pages(p, d, plan, n, true, nullptr, on.sms);
}

void pages_free(const b200_pages & p, const int32_t * slots, int n) {
    const Pages d = checked(p, false);
    need(n >= 0 && n <= (1 << 24), "pages_free: from 0 to 2^24 slots");
    need(slots || n == 0, "pages_free: null pointer");
    On on(p.device);
    heed_waits(p.device);
    if (n) launch(k_pages_free, dim3((n + 7) / 8), 256, 0, p.stream, false, 1, d, slots, n);
}

void pages_compact(const b200_pages & p, int32_t * live, void * work, int64_t work_bytes) {
    const Pages d = checked(p, true);
    need(live, "pages_compact: null pointer");
    check_work(work, work_bytes, pages_workspace(p, p.n_pages));
    On on(p.device);
    heed_waits(p.device);
    static Limits set;
    const size_t smem = words_bytes(p.n_pages);
    allow_smem(k_pages_compact, p.device, set);
    int32_t * plan = static_cast<int32_t *>(work);
    launch(k_pages_compact, dim3(1), PG_THREADS, smem, p.stream, false, 1, d, live, plan);
    move_pages(p, d, plan, p.n_pages, false, plan + PLAN_HEAD + 2 * (size_t) p.n_pages, on.sms);
}

void pages_copy(const b200_pages & p, const int32_t * src, const int32_t * dst, int n, int32_t * status, void * work, int64_t work_bytes) {
    const Pages d = checked(p, true);
    need(n >= 0 && n <= p.n_pages, "pages_copy: from 0 to n_pages pairs");
    need(status && ((src && dst) || n == 0), "pages_copy: null pointer");
    check_work(work, work_bytes, pages_workspace(p, n));
    On on(p.device);
    heed_waits(p.device);
    static Limits set;
    const size_t smem = words_bytes(p.n_pages);
    allow_smem(k_pages_check_copy, p.device, set);
    int32_t * plan = static_cast<int32_t *>(work);
    launch(k_pages_check_copy, dim3(1), PG_THREADS, smem, p.stream, false, 1, d, src, dst, n, status, plan);
    move_pages(p, d, plan, n, true, nullptr, on.sms);
}

void sample_rows(int device, void * stream, int dtype, const void * logits, int64_t row_stride, int n_rows, int n_vocab, const float * u, const float * temperature, const int32_t * top_k,
                 const float * top_p, const float * min_p, int32_t * ids, float * logprobs) {
    check_dtype(dtype, true);
    need(n_vocab >= 1 && n_vocab <= SA_MAX_VOCAB, "sample: from 1 to 2^18 logits a row (got " + std::to_string(n_vocab) + ")");
    need(n_rows >= 0 && n_rows <= (1 << 20), "sample: from 0 to 2^20 rows");
    need(row_stride >= n_vocab || n_rows <= 1, "sample: row_stride is n_vocab at least");
    need(n_rows == 0 || (logits && u && ids && aligned(logits, size_of(dtype))), "sample: null pointer");
    On on(device);
    heed_waits(device);
    if (n_rows == 0) return;
    SampleArgs a = {logits, row_stride, n_rows, n_vocab, 0, u, temperature, top_p, min_p, top_k, ids, logprobs};
    // slices of 64 KB at most, so that two blocks share an SM; smaller ones while rows leave SMs without a block and a slice has work for its threads. Mixed rows, us: 16 of 128 256 logits
    // by 8 blocks 32, by 4 48; 48 of them 45 and 56; 32 of 32 000 by 4 23, by 2 29; one of 4000 by one block 7.3, by two 7.8
    int cluster = 1;
    while (cluster < SA_MAX_CLUSTER && ((int64_t) n_vocab * size_of(dtype) > 65536ll * cluster || (n_rows * cluster < on.sms && n_vocab >= 8192 * cluster))) cluster *= 2;
    a.slice = ((n_vocab + cluster - 1) / cluster + 7) / 8 * 8;
    if (dtype == B200_DTYPE_F32) sample_as<float>(a, cluster, device, stream);
    else if (dtype == B200_DTYPE_BF16) sample_as<__nv_bfloat16>(a, cluster, device, stream);
    else sample_as<__half>(a, cluster, device, stream);
}

void kv4_status(int device) {
    need(device >= 0 && device < MAX_DEVICES, "no such device: " + std::to_string(device));
    heed_waits(device);
}
void kv4_drill(int polls) { drill_polls.store(std::max(0, polls)); }

}  // namespace b200
