// serve.cu — host side of the operators of a server that runs many sequences at once (serve.hpp): checks of arguments, launch shapes, launches on the caller's stream.
#include "serve_host.cuh"
#include "serve_attn.cuh"
#include "serve_prompt.cuh"
#include "serve_pages.cuh"
#include "serve_sample.cuh"

namespace b200 {
namespace {

using namespace srv;

static_assert(MAX_SEQ == AT_MAX_SEQ, "sequences of a step");
Cache checked(const b200_kv4 & c) { return checked_cache(c, "kv4", 18 * c.head_dim); }

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
    // a pool in 16 bits: tiles of 16 tokens as well, with as many heads of keys as of values behind them
    const bool wide = p.head_dim & B200_POOL_16BIT;
    const int hd = p.head_dim & ~B200_POOL_16BIT, heads = wide ? 2 * p.n_head_kv : p.n_head_kv, tile_bytes = (wide ? 32 : 18) * hd;
    int64_t bytes = 0;
    if (pool) {
        need(hd == 64 || hd == 128, "pages: head_dim is 64 or 128, with B200_POOL_16BIT of a pool in 16 bits (got " + std::to_string(p.head_dim) + ")");
        need(p.n_head_kv >= 1 && p.n_head_kv <= 1024 && p.n_layer >= 1 && p.n_layer <= 65536, "pages: n_head_kv from 1 to 1024, n_layer from 1 to 65536");
        bytes = (int64_t) heads * p.page_tokens / 16 * tile_bytes;
        need(p.pool && aligned(p.pool, 16), "pages: the pool starts on 16 bytes");
        need(p.page_stride >= bytes && p.page_stride % 16 == 0 && p.layer_stride % 16 == 0 && (p.n_layer == 1 || p.layer_stride >= bytes), "pages: strides hold a page and are multiples of 16 bytes");
    }
    return Pages{p.table, p.table_stride, p.n_slots, p.max_pages, p.held, p.refs, p.n_pages, log2_of(p.page_tokens), static_cast<uint8_t *>(p.pool), p.layer_stride, p.page_stride,
                 p.n_layer, heads, tile_bytes};
}
size_t words_bytes(int n) { return (size_t) ((n + 31) / 32) * 4; }
void move_pages(const b200_pages & p, const Pages & d, const int32_t * plan, int n, bool parts, const int32_t * moved_to, int sms) {
    launch(k_pages_move, dim3(sms * 4), 256, 0, p.stream, true, 1, d, plan, n, parts, moved_to);
}

template <typename T, bool VERIFY> void sample_as(const std::conditional_t<VERIFY, VerifyArgs, SampleArgs> & a, int cluster, int device, void * stream) {
    static Limits set;
    const size_t smem = SA_FIXED + ((size_t) a.slice * sizeof(T) + 15) / 16 * 16;
    const auto kernel = k_sample<T, VERIFY>;
    allow_smem(kernel, device, set);
    launch(kernel, dim3((unsigned) (a.n_rows * cluster)), SA_THREADS, smem, stream, VERIFY, cluster, a);
}

template <bool VERIFY, typename A> void sample_all(A & a, int dtype, const On & on, void * stream) {
    // slices of 64 KB at most, so that two blocks share an SM; smaller ones while rows leave SMs without a block and a slice has work for its threads. Mixed rows, us: 16 of 128 256 logits
    // by 8 blocks 32, by 4 48; 48 of them 45 and 56; 32 of 32 000 by 4 23, by 2 29; one of 4000 by one block 7.3, by two 7.8
    int cluster = 1;
    while (cluster < SA_MAX_CLUSTER && ((int64_t) a.n_vocab * size_of(dtype) > 65536ll * cluster || (a.n_rows * cluster < on.sms && a.n_vocab >= 8192 * cluster))) cluster *= 2;
    a.slice = ((a.n_vocab + cluster - 1) / cluster + 7) / 8 * 8;
    if constexpr (VERIFY) {
        if ((int64_t) a.n_rows * cluster <= 2 * on.sms) a.order = a.ended = nullptr;      // all rows are on the card at once
        else launch(k_verify_order, dim3((unsigned) ((a.n_rows + VO_THREADS - 1) / VO_THREADS)), VO_THREADS, 4 * (2 * (size_t) a.n_seq + 1), stream, true, 1, a);
    }
    if (dtype == B200_DTYPE_F32) sample_as<float, VERIFY>(a, cluster, on.device, stream);
    else if (dtype == B200_DTYPE_BF16) sample_as<__nv_bfloat16, VERIFY>(a, cluster, on.device, stream);
    else sample_as<__half, VERIFY>(a, cluster, on.device, stream);
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

void pages_plan(const b200_pages & p, const int32_t * slots, const int32_t * counts, int n, int n_rows, int32_t * first, int32_t * positions, int32_t * places, int32_t * status) {
    const Pages d = checked(p, false);
    need(n >= 0 && n <= PG_MAX_N, "pages_plan: from 0 to " + std::to_string(PG_MAX_N) + " sequences");
    need(n_rows >= 0 && n_rows <= (1 << 24), "pages_plan: from 0 to 2^24 rows");
    need((counts || n == 0) && first && status && ((positions && places) || n_rows == 0), "pages_plan: null pointer");
    need(slots || n <= p.n_slots, "pages_plan: more sequences than slots");
    On on(p.device);
    heed_waits(p.device);
    static Limits set;
    const bool apart = n_rows > PLAN_ROWS;
    const size_t smem = words_bytes(p.n_slots) + plan_bytes(n), places_smem = 4 * ((size_t) 3 * n + 1);
    allow_smem(k_pages_plan, p.device, set);
    launch(k_pages_plan, dim3(1), PG_THREADS, smem, p.stream, true, 1, d, slots, counts, n, n_rows, first, positions, places, status, !apart);
    static Limits places_set;
    if (apart) allow_smem(k_pages_places, p.device, places_set);
    if (apart) launch(k_pages_places, dim3((unsigned) ((n_rows + 1023) / 1024)), 256, places_smem, p.stream, true, 1, d, slots, first, n, n_rows, positions, places);
}

void pages_trim(const b200_pages & p, const int32_t * slots, int n, int window, int sinks) {
    const Pages d = checked(p, false);
    need(n >= 0 && n <= (1 << 24) && (int64_t) n * ((p.max_pages + 255) / 256) <= 1ll << 33, "pages_trim: from 0 to 2^24 slots, and to 2^41 pages of their tables");
    need(slots || n == 0, "pages_trim: null pointer");
    need(window >= 0 && sinks >= 0, "pages_trim: window is a number of positions, or 0 for all; sinks is a number of positions");
    On on(p.device);
    heed_waits(p.device);
    if (n) launch(k_pages_trim, dim3((unsigned) (((int64_t) n * ((p.max_pages + 255) / 256) + 7) / 8)), 256, 0, p.stream, true, 1, d, slots, n, window, sinks);
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
    sample_all<false>(a, dtype, on, stream);
}

int64_t verify_workspace(int n_rows) {
    need(n_rows >= 0 && n_rows <= (1 << 20), "verify: from 0 to 2^20 rows");
    return 8 * (int64_t) n_rows;
}
void verify_rows(int device, void * stream, int dtype, const void * logits, int64_t row_stride, int n_rows, int n_vocab, const int32_t * ids, const int32_t * first, int n_seq, const float * u,
                 const float * accept, const float * temperature, const int32_t * top_k, const float * top_p, const float * min_p, const float * draft_probs, int64_t draft_stride,
                 int32_t * gained, int32_t * tokens, float * logprobs, void * work, int64_t work_bytes) {
    check_dtype(dtype, true);
    need(n_vocab >= 1 && n_vocab <= SA_MAX_VOCAB, "verify: from 1 to 2^18 logits a row (got " + std::to_string(n_vocab) + ")");
    need(n_rows >= 0 && n_rows <= (1 << 20), "verify: from 0 to 2^20 rows");
    need(n_seq >= 0 && n_seq <= MAX_SEQ, "verify: from 0 to 4096 sequences");
    need(row_stride >= n_vocab || n_rows <= 1, "verify: row_stride is n_vocab at least");
    need(!draft_probs || draft_stride >= n_vocab || n_rows <= 1, "verify: draft_stride is n_vocab at least");
    need(first && (gained || n_seq == 0), "verify: null pointer");
    need(n_rows == 0 || (logits && ids && u && accept && tokens && logprobs && aligned(logits, size_of(dtype))), "verify: null pointer");
    if (n_rows) check_work(work, work_bytes, verify_workspace(n_rows));
    On on(device);
    heed_waits(device);
    int32_t * order = static_cast<int32_t *>(work);
    VerifyArgs a = {{logits, row_stride, n_rows, n_vocab, 0, u, temperature, top_p, min_p, top_k, tokens, logprobs}, ids, first, n_seq, accept, draft_probs, draft_stride, gained, order, order + n_rows};
    if (n_rows) sample_all<true>(a, dtype, on, stream);
    if (n_seq) launch(k_verify_ends<128>, dim3((unsigned) ((n_seq + 3) / 4)), 128, 0, stream, true, 1, a);
}

void kv4_status(int device) {
    need(device >= 0 && device < MAX_DEVICES, "no such device: " + std::to_string(device));
    heed_waits(device);
}
void kv4_drill(int polls) { drill_polls.store(std::max(0, polls)); }

}  // namespace b200
