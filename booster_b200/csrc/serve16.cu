// serve16.cu — host side of the 16-bit paged cache (serve.hpp): checks of arguments, launch shapes, launches on the caller's stream.
#include "serve_host.cuh"
#include "serve_kv16_prompt.cuh"

namespace b200 {
namespace {

using namespace srv;

Cache checked(const b200_kv4 & c) { return checked_cache(c, "kv16", 64 * c.head_dim); }

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
CUtensorMap map_of(bool bf16, int n, const void * base, const cuuint64_t * dims, const cuuint64_t * strides, const cuuint32_t * box) {
    static const auto encode = [] {
        void * fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) { cudaGetLastError(); fn = nullptr; }
        return reinterpret_cast<EncodeTiled>(fn);
    }();
    need(encode, "the driver has no cuTensorMapEncodeTiled");
    CUtensorMap m;
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    const CUresult r = encode(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, n, const_cast<void *>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed: " + std::to_string((int) r));
    return m;
}
// boxes of `tokens` tokens and 64 dims of a KV head of a page, of keys and values at once or of one of them
CUtensorMap pool_map(const b200_kv4 & c, bool bf16, int tokens, int sides) {
    const cuuint64_t row = (cuuint64_t) c.head_dim * 2, head = row * c.page_tokens, side = head * c.n_head_kv;
    const cuuint64_t dims[5] = {(cuuint64_t) c.head_dim, (cuuint64_t) c.page_tokens, (cuuint64_t) c.n_head_kv, 2, (cuuint64_t) c.n_pages}, strides[4] = {row, head, side, (cuuint64_t) c.page_stride};
    const cuuint32_t box[5] = {64, (cuuint32_t) tokens, 1, (cuuint32_t) sides, 1};
    return map_of(bf16, 5, c.pool, dims, strides, box);
}

template <typename S, typename T> void append_as(const b200_kv4 & c, const Cache & d, const void * k, int64_t kr, int64_t kh, const void * v, int64_t vr, int64_t vh) {
    const Row16Src<S> src = {static_cast<const S *>(k), kr, kh, static_cast<const S *>(v), vr, vh, aligned(k, 16) && aligned(v, 16) && !((kr | kh | vr | vh) & (16 / (int64_t) sizeof(S) - 1))};
    const int per = 256 / c.head_dim, parts = (c.n_head_kv + per - 1) / per;
    const auto rows = [&](auto kernel) { launch(kernel, dim3((unsigned) (((int64_t) c.n_rows * parts + 7) / 8)), 256, 0, c.stream, true, 1, d, src, parts); };
    c.head_dim == 128 ? rows(k_kv16_append<S, T, 128>) : rows(k_kv16_append<S, T, 64>);
}
template <typename T> void append_to(const b200_kv4 & c, const Cache & d, int dtype, const void * k, int64_t kr, int64_t kh, const void * v, int64_t vr, int64_t vh) {
    if (dtype == B200_DTYPE_F32) append_as<float, T>(c, d, k, kr, kh, v, vr, vh);
    else if (dtype == B200_DTYPE_BF16) append_as<__nv_bfloat16, T>(c, d, k, kr, kh, v, vr, vh);
    else append_as<__half, T>(c, d, k, kr, kh, v, vr, vh);
}

// columns of a unit: 8 or 16 of one warp, in one launch also 32 or 64 of two or four that share what is read
int attend_cols(int group, int max_rows) { const int64_t n = (int64_t) group * max_rows; return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : 128; }
size_t attend_before_bytes(int n_seq) { return ((size_t) (n_seq + 2) * 8 + 255) / 256 * 256; }
size_t attend_columns(int cols, int sms) { return 2 * (size_t) sms * A16_WARPS * cols; }      // of all pieces' partial results
size_t attend_bytes(int n_seq, int head_dim, int cols, int sms) { return attend_before_bytes(n_seq) + attend_columns(cols, sms) * (head_dim + 2) * 4; }
struct Few { CUtensorMap map; int * err; uint32_t polls; int boxes, cluster, device, sms; void * stream; };
template <int HD, int NT, int CW, typename T> void unit_as(const AttendArgs & a, const Few & f) {
    static Limits set;
    const auto kernel = k_kv16_attend_unit<HD, NT, CW, T>;
    allow_smem(kernel, f.device, set);
    launch(kernel, dim3((unsigned) (a.c.n_seq * a.c.n_kv * f.cluster)), A16_WARPS * 32, 1024 + a16_ring_bytes(HD), f.stream, true, f.cluster, a, f.map, f.err, f.polls, f.boxes);
}
template <int HD, int NT, typename T> void attend_as(const AttendArgs & a, const Few & f) {
    if (f.cluster) return unit_as<HD, NT, 1, T>(a, f);
    static Limits set;
    const auto kernel = k_kv16_attend<HD, NT, T>;
    allow_smem(kernel, f.device, set);
    launch(kernel, dim3(f.sms), A16_WARPS * 32, 1024 + a16_ring_bytes(HD) + (size_t) (a.c.n_seq + 1) * 8, f.stream, true, 1, a, f.map, f.err, f.polls, f.boxes);
    // warps that add a unit's parts, where it has so many on average, 16 / 4 / 1, us a call: one of 20 000 (74) 21.9 / 25.0 / 29.9, 2 of 30 000 (37) 47.6 / 49.8 / 52.6, 4 of 12 000 (18) 39.9 / 40.1 / 42.0, 16 of 20 000 (2 heads of 64,
    // 18) 34.7 / 34.3 / 35.9, 12 of 3000 (6) 33.8 / 32.7 / 32.0, 48 ragged (1.5) 83.8 / 75.9 / 74.4, 200 of 500 112 / 83 / 77. What beginning a unit costs (AT_OVER, in pairs of 4-bit tiles 3) is 3 steps here too: 48 ragged 79, 77, 74,
    // 75, 74, 74 with 0, 1, 2, 3, 4, 6, four rows each 102, 89, 84, 81, 81, 80
    const int64_t items = (int64_t) a.c.n_rows * a.c.n_kv * a.group, parts = (int64_t) f.sms * A16_WARPS / ((int64_t) a.c.n_seq * a.c.n_kv);
    if (parts > 32) launch(k_kv4_join<HD, NT, T, 16>, dim3((unsigned) items), 512, 0, f.stream, true, 1, a);
    else if (parts > 8) launch(k_kv4_join<HD, NT, T, 4>, dim3((unsigned) items), 128, 0, f.stream, true, 1, a);
    else launch(k_kv4_join<HD, NT, T, 1>, dim3((unsigned) ((items + 7) / 8)), 256, 0, f.stream, true, 1, a);
}
template <int HD, typename T> void attend_few(const AttendArgs & a, const Few & f, int cols) {
    if (cols == 8) attend_as<HD, 1, T>(a, f);
    else if (cols == 16) attend_as<HD, 2, T>(a, f);
    else if (cols == 32) unit_as<HD, 2, 2, T>(a, f);
    else unit_as<HD, 2, 4, T>(a, f);
}
// clusters of so many blocks (2, 4 or 8) that the card holds at once: a cluster stands within one group of SMs, and those are not all of a size that 8 goes into (two blocks an SM with heads of 64). All
// of k_kv16_attend_unit's forms for a head_dim have the same of it
int clusters_at_once(int head_dim, int cluster, int device) {
    static std::atomic<int> known[2][A16_CLUSTER + 1][MAX_DEVICES];       // one more than there are
    static Limits set[2];
    const bool wide = head_dim == 128;
    std::atomic<int> & n = known[wide][cluster][device];
    if (const int have = n.load()) return have - 1;
    const auto kernel = wide ? k_kv16_attend_unit<128, 1, 1, __nv_bfloat16> : k_kv16_attend_unit<64, 1, 1, __nv_bfloat16>;
    allow_smem(kernel, device, set[wide]);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension; at.val.clusterDim.x = cluster; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
    cfg.gridDim = dim3(cluster); cfg.blockDim = dim3(A16_WARPS * 32); cfg.dynamicSmemBytes = 1024 + a16_ring_bytes(head_dim); cfg.attrs = &at; cfg.numAttrs = 1;
    int got = 0;
    cu(cudaOccupancyMaxActiveClusters(&got, kernel, &cfg), "cudaOccupancyMaxActiveClusters");
    n.store(got + 1);
    return got;
}
// blocks of a cluster a unit where one launch does: all clusters stand on the card at once (in two waves two sequences of 2000 take 13.7 us for 9.0 by half as large ones), and the longest sequence that
// the table (or the window) allows gives each warp (or group of warps) at most so many steps of 32 tokens. 0: a line of pieces and a join, or tcgen05. It goes by the table's width because the host does not
// know the lengths: under a table for long contexts short sequences take the other form. One launch / two, us a call among others, 8 KV heads of 128: one sequence of 333 (1 step) 5.6 / 8.5, of 8000 (8)
// 12.2 / 14.2, of 16 000 (16) 18.7 / 18.9; 2 of 2000 (4) 9.0 / 12.1, of 8000 (16) 18.5 / 19.2; 16 of 200 (2) 7.2 / 11.4, of 1000 (8) 14.9 / 18.8; 61 of 1000 (2 heads of 64, 8) 10.1 / 13.7. More columns,
// one launch / tcgen05: 20 columns, one of 1000 (2) 8.9 / 14.7, of 3900 (8) 15.0 / 19.9, 2 of 1900 (8) 15.6 / 17.2, 8 of 1000 (8) 16.5 / 20.2; 64 columns, one of 1000 (4) 12.5 / 14.7, of 1900 (8) 17.0 / 17.9, 4 of 500 (5) 16.2 / 16.4, but 2 of
// 1000 (8, by 4 blocks) 19.5 / 16.1
int unit_steps(int cols, int cluster) { return cols <= 16 ? 16 : cols <= 32 || cluster == A16_CLUSTER ? 8 : 4; }
int unit_cluster(const b200_kv4 & c, int cols, int window, int sinks, const On & on) {
    const int64_t units = (int64_t) c.n_seq * c.n_head_kv, room = (int64_t) on.sms * (c.head_dim == 64 ? 2 : 1);
    if (cols > 64 || units > room) return 0;
    int64_t tokens = (int64_t) c.max_pages * c.page_tokens;
    if (window > 0) tokens = std::min(tokens, (int64_t) window + std::min<int64_t>(sinks, tokens) + 128);
    int cluster = A16_CLUSTER;
    while (cluster > 1 && units > clusters_at_once(c.head_dim, cluster, on.device)) cluster /= 2;
    return (tokens + 31) / 32 <= (int64_t) unit_steps(cols, cluster) * (cols <= 16 ? A16_WARPS : 64 / cols) * cluster ? cluster : 0;
}

template <int HD, typename T> void prompt_as(const PromptArgs & p, const CUtensorMap & map, const CUtensorMap & q_map, bool by_box, int64_t entries, int device, int sms, void * stream) {
    static Limits set;
    const auto kernel = k_kv16_prompt<HD, T>;
    allow_smem(kernel, device, set);
    launch(k_kv16_plan, dim3(1), 1024, (size_t) (p.a.c.n_seq + 1) * 4, stream, true, 1, p, sms);
    launch(kernel, dim3(sms), P16_THREADS, Prompt16Smem<HD>::BYTES, stream, true, 1, p, map, q_map, by_box);
    launch(k_kv16_prompt_join<HD, T>, dim3((unsigned) (entries * (PR_COLS / 32)), (unsigned) p.a.c.n_kv), 256, 0, stream, true, 1, p);
}

void check_heads(const b200_kv4 & c, int n_head, int max_rows) {
    need(n_head >= c.n_head_kv && n_head % std::max(1, c.n_head_kv) == 0 && (int64_t) c.n_rows * n_head <= (1 << 30), "n_head is a multiple of n_head_kv, and rows x heads up to 2^30");
    need(max_rows >= 1 && max_rows <= (1 << 24), "max_rows is the largest number of rows of a sequence");
}

}  // namespace

void kv16_append(const b200_kv4 & c, int pool_dtype, int dtype, const void * k, int64_t k_row, int64_t k_head, const void * v, int64_t v_row, int64_t v_head) {
    const Cache d = checked(c);
    check_dtype(pool_dtype, false);
    check_dtype(dtype, true);
    need(c.n_rows == 0 || (k && v && aligned(k, size_of(dtype)) && aligned(v, size_of(dtype))), "k and v are pointers to whole entries");
    On on(c.device);
    heed_waits(c.device);
    if (c.n_seq == 0 || c.n_rows == 0) return;
    pool_dtype == B200_DTYPE_BF16 ? append_to<__nv_bfloat16>(c, d, dtype, k, k_row, k_head, v, v_row, v_head) : append_to<__half>(c, d, dtype, k, k_row, k_head, v, v_row, v_head);
}

int64_t kv16_attention_workspace(const b200_kv4 & c, int n_head, int max_rows) {
    checked(c);
    check_heads(c, n_head, max_rows);
    On on(c.device);
    const int group = n_head / c.n_head_kv, cols = attend_cols(group, max_rows);
    if (unit_cluster(c, cols, 0, 0, on)) return 0;       // (a window asks for no more)
    return cols > 16 ? prompt_work(c, group, on.sms).bytes : (int64_t) attend_bytes(c.n_seq, c.head_dim, cols, on.sms);
}

void kv16_attention(const b200_kv4 & c, int dtype, const void * q, int64_t q_row, int64_t q_head, int n_head, float scale, int window, int sinks, int max_rows, void * out, void * work,
                    int64_t work_bytes) {
    AttendArgs a = {};
    a.c = checked(c);
    check_dtype(dtype, false);
    check_heads(c, n_head, max_rows);
    need(c.n_rows == 0 || (q && out && aligned(q, 2) && aligned(out, 16)), "q points to whole entries, out starts on 16 bytes");
    need(std::isfinite(scale), "scale is a finite number");
    need(window >= 0 && sinks >= 0, "window is a number of positions, or 0 for all; sinks is a number of positions");
    On on(c.device);
    heed_waits(c.device);
    if (c.n_seq == 0 || c.n_rows == 0) return;
    a.q = q; a.q_row = q_row; a.q_head = q_head; a.out = out;
    a.q_whole = aligned(q, 16) && !((q_row | q_head) & 7);
    a.group = n_head / c.n_head_kv;
    a.scale_log2 = scale * 1.44269504088896341f;
    a.window = window;
    a.sinks = window > 0 ? sinks : 0;
    uint8_t * w = static_cast<uint8_t *>(work);
    const bool bf16 = dtype == B200_DTYPE_BF16;
    int * err = wait_word(c.device);
    const int drill = drill_polls.load(), never = 1 << 19;       // (more arrivals than come)
    const uint32_t polls = drill ? (uint32_t) drill : WAIT_POLLS;
    // up to 16 columns of a sequence (rows x query heads of a KV head) are one warp's; more are worth tcgen05's plan and join where one launch does not do
    const int cols = attend_cols(a.group, max_rows), cluster = unit_cluster(c, cols, window, a.sinks, on);
    if (cols > 16 && !cluster) {
        const PromptWork at = prompt_work(c, a.group, on.sms);
        check_work(work, work_bytes, at.bytes);
        const int64_t n = prompt_entries(c, a.group);
        // 128 columns as one box: whole rows of a group, rows and heads at distances that a tensor map can have
        const bool by_box = a.q_whole && 128 % a.group == 0 && q_head > 0 && (q_row > 0 || c.n_rows == 1) && q_row < (1ll << 38) && q_head < (1ll << 38);
        PromptArgs p = {a, (int) n, reinterpret_cast<Entry *>(w + at.entries), reinterpret_cast<int *>(w + at.first), err, polls, drill ? never : by_box ? 1 : 4};
        p.a.before = reinterpret_cast<long long *>(w);
        p.a.ml = reinterpret_cast<float *>(w + at.ml);
        p.a.part = reinterpret_cast<float *>(w + at.part);
        const CUtensorMap map = pool_map(c, bf16, std::min(c.page_tokens, PR_KV), 1);
        CUtensorMap q_map = {};
        if (by_box) {
            const cuuint64_t dims[3] = {(cuuint64_t) c.head_dim, (cuuint64_t) n_head, (cuuint64_t) c.n_rows}, strides[2] = {(cuuint64_t) q_head * 2, (cuuint64_t) (c.n_rows > 1 ? q_row : 8) * 2};
            const cuuint32_t box[3] = {64, (cuuint32_t) a.group, (cuuint32_t) (128 / a.group)};
            q_map = map_of(bf16, 3, q, dims, strides, box);
        }
        const auto as = [&](auto run) { run(p, map, q_map, by_box, n, c.device, on.sms, c.stream); };
        if (bf16) c.head_dim == 128 ? as(prompt_as<128, __nv_bfloat16>) : as(prompt_as<64, __nv_bfloat16>);
        else c.head_dim == 128 ? as(prompt_as<128, __half>) : as(prompt_as<64, __half>);
        return;
    }
    if (!cluster) check_work(work, work_bytes, (int64_t) attend_bytes(c.n_seq, c.head_dim, cols, on.sms));
    a.before = reinterpret_cast<long long *>(w);
    a.ml = reinterpret_cast<float *>(w + attend_before_bytes(c.n_seq));
    a.part = a.ml + attend_columns(cols, on.sms) * 2;
    const Few f = {pool_map(c, bf16, 16, 2), err, polls, drill ? never : 1, cluster, c.device, on.sms, c.stream};
    if (bf16) c.head_dim == 128 ? attend_few<128, __nv_bfloat16>(a, f, cols) : attend_few<64, __nv_bfloat16>(a, f, cols);
    else c.head_dim == 128 ? attend_few<128, __half>(a, f, cols) : attend_few<64, __half>(a, f, cols);
}

}  // namespace b200
