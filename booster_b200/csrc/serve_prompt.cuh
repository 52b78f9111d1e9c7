// serve_prompt.cuh — attention of prompts' portions over the 4-bit cache (sm_100a, tcgen05): many rows of a sequence.
//
// A unit of work is 256 columns of a sequence (a column is a row and a query head of one KV head) over the tiles of 128 tokens that they see. As for few rows, all units stand in one
// line that is cut evenly, here over one block per SM; k_kv4_prompt_plan lays the line out, k_kv4_prompt_join adds the parts of units that blocks shared.
//   warps 0-3, 4-7   soft-max of columns 0-127 and 128-255, a thread a column: maximum and exponentials of its row of S, P back into tensor memory in the place of S
//   warps 8-11       codes of 32 tokens each to fp16 in shared memory (exact: a scale has 8 bits, a code 4), K by rows of tokens, V by rows of dims, both with 128-byte swizzle
//   warp 12          one thread issues S = Q K^T (128 x 128 x head_dim, twice) and O += P V (P from tensor memory, 128 x head_dim x 128, twice)
// While one half's soft-max runs, the other half's products do. Tensor memory: S and P [2][128 columns], O [2][head_dim].
// Tokens of 32 stand as n = 8 c + 4 u + i for token 16 u + c + 4 i in S, P, K and V alike, and dims of 8 as 0 4 1 5 2 6 3 7 in Q and K: the orders in which a word's codes come apart.
// P is rounded to fp16 (2^-11), q scaled by a power of two into fp16's range; sums are fp32. The maximum moves when a score passes it by 2^8; O is scaled in tensor memory then.
// Every wait on an mbarrier is bounded: on a timeout the block raises *err, skips what is left and frees its tensor memory.
#pragma once
#include "serve_attn.cuh"

namespace b200 {
namespace srv {

struct PromptArgs {
    AttendArgs a;                        // a.before: [entries + 1] tiles in front of each entry (a sequence's 256 columns), for all KV heads together
    int * seq_of, * entry_of, * n_entries;   // [entries], [n_seq + 1], {entries, tiles of a block's piece}
    int * err;
};

constexpr int PR_COLS = 256, PR_KV = 128, PR_THREADS = 416, PR_OVER = 2;      // PR_OVER: what beginning a unit costs, in tiles
constexpr uint64_t PR_DESC = (1ull << 16) | ((uint64_t) (1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);      // K-major, 128-byte swizzle, groups of 8 rows 1024 bytes apart
__host__ __device__ constexpr uint32_t pr_idesc(int n) { return (1u << 4) | ((uint32_t) (n >> 3) << 17) | (8u << 24); }     // D f32, A and B f16, M = 128
template <int HD> struct PromptSmem {
    static constexpr int Q = 128 * HD * 2, KV = PR_KV * HD * 2;      // bytes of one half of Q, of a tile's K or V
    static constexpr int BYTES = 2 * Q + 4 * KV + 1024;              // K and V in two stages each
};

__device__ __forceinline__ void pr_wait(uint32_t bar, uint32_t parity, bool & dead) {
    for (uint32_t spins = 0; !dead; spins++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) break;
        if (spins >= (1u << 22)) dead = true;
    }
}
__device__ __forceinline__ void pr_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory"); }
__device__ __forceinline__ void pr_commit(uint32_t bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory"); }
__device__ __forceinline__ void pr_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pr_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ bool pr_elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void pr_mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" :: "r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void pr_mma_ts(uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" :: "r"(d), "r"(a), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void pr_ld32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
                   "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
                   "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(at) : "memory");
}
// the registers hold what was loaded behind this
__device__ __forceinline__ void pr_ld32_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]),
                   "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]) :: "memory");
}
__device__ __forceinline__ void pr_st32(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
                 :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                    "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
                    "r"(r[30]), "r"(r[31]), "r"(at) : "memory");
}
__device__ __forceinline__ void pr_st16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
                 :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
                    "r"(r[15]), "r"(at) : "memory");
}
__device__ __forceinline__ void pr_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pr_st_shared(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// tiles of 128 tokens that the columns of an entry see, one at least
__device__ __forceinline__ Span prompt_span(const Cache & c, const Seq & q, int group, int window, int ct) {
    const int a = ct * PR_COLS / group, b = min(q.count - 1, (ct * PR_COLS + PR_COLS - 1) / group);
    const int last = min(q.held + b, (c.max_pages << c.page_log2) - 1), first = window > 0 ? max(0, q.held + a - window + 1) : 0;
    Span s;
    s.lo = first / PR_KV;
    s.n = q.slot < 0 || last < first ? 1 : last / PR_KV - s.lo + 1;
    return s;
}

// one block: the line of entries
__global__ void __launch_bounds__(1024) k_kv4_prompt_plan(const PromptArgs p, int n_blocks) {
    __shared__ long long sums[32];
    __shared__ int counts[32];
    const Cache & c = p.a.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int each = (c.n_seq + 1023) / 1024, s0 = min(c.n_seq, tid * each), s1 = min(c.n_seq, s0 + each);
    long long tiles = 0;
    int entries = 0;
    for (int s = s0; s < s1; s++) {
        const Seq q = seq_at(c, s);
        const int n = col_tiles(q, p.a.group, PR_COLS);
        entries += n;
        for (int ct = 0; ct < n; ct++) tiles += (long long) c.n_kv * (prompt_span(c, q, p.a.group, p.a.window, ct).n + PR_OVER);
    }
    long long up = tiles;
    int upe = entries;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, up, d);
        const int y = __shfl_up_sync(0xffffffffu, upe, d);
        if (lane >= d) { up += x; upe += y; }
    }
    if (lane == 31) { sums[warp] = up; counts[warp] = upe; }
    __syncthreads();
    long long at = up - tiles, total = 0;
    int e = upe - entries, all = 0;
    for (int w = 0; w < 32; w++) {
        if (w < warp) { at += sums[w]; e += counts[w]; }
        total += sums[w]; all += counts[w];
    }
    for (int s = s0; s < s1; s++) {
        const Seq q = seq_at(c, s);
        const int n = col_tiles(q, p.a.group, PR_COLS);
        p.entry_of[s] = e;
        for (int ct = 0; ct < n; ct++, e++) {
            p.seq_of[e] = s;
            p.a.before[e] = at;
            at += (long long) c.n_kv * (prompt_span(c, q, p.a.group, p.a.window, ct).n + PR_OVER);
        }
    }
    if (tid == 0) {
        p.a.before[all] = total;
        p.entry_of[c.n_seq] = all;
        p.n_entries[0] = all;
        p.n_entries[1] = (int) max(1ll, (total + n_blocks - 1) / n_blocks);
    }
}

// a piece of one unit
struct Segment { Seq q; Span sp; int ct, head, t0, t1, halves; bool run; };

// P's columns hold tokens in this order (of 32)
__host__ __device__ constexpr int token_of(int col) { return 16 * (col >> 2 & 1) + (col >> 3) + 4 * (col & 3); }

template <int HD, typename T>
__global__ void __launch_bounds__(PR_THREADS, 1) k_kv4_prompt(const PromptArgs p) {
    constexpr int NB = HD / 32, TILE = 18 * HD, QB = PromptSmem<HD>::Q, KVB = PromptSmem<HD>::KV, SUB = 128 * 128;      // SUB: 128 rows of 128 bytes
    extern __shared__ uint8_t pr_raw[];
    __shared__ __align__(8) uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2];
    __shared__ uint32_t tmem_s;
    const AttendArgs & a = p.a;
    const Cache & c = a.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t smem = (smem_at(pr_raw) + 1023u) & ~1023u, q_s = smem, k_s = q_s + 2 * QB, v_s = k_s + 2 * KVB;
    if (tid == 0) {
        const auto init = [](uint64_t * b, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(smem_at(b)), "r"(n) : "memory"); };
        for (int i = 0; i < 2; i++) { init(&q_full[i], 4); init(&k_full[i], 4); init(&v_full[i], 4); init(&k_empty[i], 1); init(&v_empty[i], 1); init(&s_full[i], 1); init(&p_full[i], 4); init(&o_full[i], 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(smem_at(&tmem_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pr_fence_before();
    __syncthreads();
    pr_fence_after();
    const uint32_t tmem = tmem_s, t_s = tmem, t_o = tmem + 256;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int entries = p.n_entries[0], per = p.n_entries[1];
    const long long begin = (long long) blockIdx.x * per, end = min(a.before[entries], begin + per);
    // the segments of this block's piece, the same for every warp
    const auto segment = [&](long long & at) {
        Segment g;
        int e = 0, n = entries;
        while (n > 1) {                                            // the last entry that begins at or before `at`, 32 places at a time
            const int step = (n + 31) >> 5, i = e + lane * step;
            const unsigned m = __ballot_sync(0xffffffffu, lane * step < n && a.before[min(i, entries - 1)] <= at);
            const int k = m ? 31 - __clz(m) : 0;
            e += k * step;
            n = min(step, n - k * step);
        }
        const int s = p.seq_of[e];
        g.q = seq_at(c, s);
        g.ct = e - p.entry_of[s];
        g.sp = prompt_span(c, g.q, a.group, a.window, g.ct);
        const long long x = at - a.before[e];
        const int len = g.sp.n + PR_OVER, from = (int) (x % len), to = (int) min((long long) len, from + (end - at));
        g.head = (int) (x / len);
        g.t0 = max(0, from - PR_OVER);
        g.t1 = to - PR_OVER;
        g.run = g.t1 > 0;
        g.halves = g.q.count * a.group - g.ct * PR_COLS > 128 ? 2 : 1;
        at += to - from;
        return g;
    };
    bool dead = false;
    if (warp < 8) {
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;          // of the half
        const uint32_t lanes = (uint32_t) ((warp & 3) * 32) << 16, my_s = t_s + lanes + half * 128, my_o = t_o + lanes + half * HD;
        int n_s = 0;                                                       // tiles of this half so far
        for (long long at = begin; at < end;) {
            const Segment g = segment(at);
            if (!g.run) continue;
            const int col = g.ct * PR_COLS + half * 128 + row, i = col / a.group, h = g.head * a.group + col - i * a.group;
            const bool in = i < g.q.count;
            if (half >= g.halves) continue;
            float factor;
            {
                // the column's query, scaled by a power of two to at most 2^14, dims of eight as 0 4 1 5 2 6 3 7
                const T * src = static_cast<const T *>(a.q) + (in ? (g.q.begin + i) * a.q_row + h * a.q_head : 0);
                const auto load = [&](int m) {
                    Eight<T> f = {};
                    if (in) {
                        if (a.q_whole) f = *reinterpret_cast<const Eight<T> *>(src + 8 * m);
                        else for (int j = 0; j < 8; j++) f.v[j] = src[8 * m + j];
                    }
                    return f;
                };
                float top = 0.f;
#pragma unroll 4
                for (int m = 0; m < HD / 8; m++) {
                    const Eight<T> f = load(m);
#pragma unroll
                    for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(to_f(f.v[j])));
                }
                const int e = min(126, max(-126, 140 - (int) (__float_as_uint(top) >> 23)));
                float up = top > 0.f && top < INFINITY ? __uint_as_float((uint32_t) (127 + e) << 23) : 1.f;
                factor = fmaxf(fabsf(a.scale_log2) / up, 1.2e-38f);           // (never 0: it meets the -infinity of what is masked)
                if (a.scale_log2 < 0.f) up = -up;
#pragma unroll 4
                for (int m = 0; m < HD / 8; m++) {
                    const Eight<T> f = load(m);
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) w[j] = as_u(__floats2half2_rn(to_f(f.v[j]) * up, to_f(f.v[j + 4]) * up));
                    pr_st_shared(q_s + half * QB + (m >> 3) * SUB + row * 128 + (((m & 7) ^ (row & 7)) << 4), w[0], w[1], w[2], w[3]);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) pr_arrive(smem_at(&q_full[half]));
            // whether every page of the piece is there; where not, each tile's are looked up again
            bool whole = g.q.slot >= 0;
            {
                const int a0 = ((g.sp.lo + g.t0) * PR_KV) >> c.page_log2, a1 = min((g.sp.lo + g.t1) * PR_KV - 1, g.q.held + g.q.count - 1) >> c.page_log2;
                for (int x = a0 + lane; x <= a1; x += 32) whole = whole && page_at(c, g.q.slot, x << c.page_log2) >= 0;
                whole = __all_sync(0xffffffffu, whole);
            }
            const int row_lo = g.ct * PR_COLS / a.group, row_hi = min(g.q.count - 1, (g.ct * PR_COLS + PR_COLS - 1) / a.group);
            const int all_see_hi = g.q.held + row_lo, all_see_lo = a.window > 0 ? g.q.held + row_hi - a.window + 1 : 0;
            const int top_pos = in ? g.q.held + i : -1, low_pos = a.window > 0 ? top_pos - a.window : -1;      // sees low_pos < position <= top_pos
            float m = -INFINITY, l = 0.f, base = 0.f, limit = -INFINITY;
            for (int t = g.t0; t < g.t1; t++, n_s++) {
                const int pos = (g.sp.lo + t) * PR_KV;
                const bool edge = !whole || pos + PR_KV - 1 > all_see_hi || pos < all_see_lo;
                unsigned there = 0xffu;                                    // tiles of 16 tokens that have a page
                if (!whole) there = __ballot_sync(0xffffffffu, lane < 8 && page_at(c, g.q.slot, pos + 16 * (lane & 7)) >= 0);
                const auto hide = [&](uint32_t (&r)[32], int ch) {
                    const int hi = top_pos - pos - 32 * ch, lo = low_pos - pos - 32 * ch;
#pragma unroll
                    for (int x = 0; x < 32; x++)
                        if (token_of(x) > hi || token_of(x) <= lo || !(there >> (2 * ch + (x >> 2 & 1)) & 1)) r[x] = 0xff800000u;
                };
                pr_wait(smem_at(&s_full[half]), (uint32_t) (n_s & 1), dead);
                __syncwarp();
                pr_fence_after();
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int ch = 0; ch < 4; ch++) {
                    uint32_t r[32];
                    pr_ld32(my_s + 32 * ch, r);
                    pr_ld32_wait(r);
                    if (edge) hide(r, ch);
#pragma unroll
                    for (int x = 0; x < 32; x += 2) { x0 = fmaxf(x0, __uint_as_float(r[x])); x1 = fmaxf(x1, __uint_as_float(r[x + 1])); }
                }
                const float high = fmaxf(x0, x1), score = high == -INFINITY ? high : high * factor;
                if (__any_sync(0xffffffffu, score > limit)) {
                    const float top = fmaxf(m, score), down = top > m ? exp2_fast(m - top) : 1.f;
                    if (t > g.t0 && __any_sync(0xffffffffu, down != 1.f)) {
                        pr_wait(smem_at(&o_full[half]), (uint32_t) ((n_s - 1) & 1), dead);
                        __syncwarp();
                        pr_fence_after();
#pragma unroll
                        for (int ch = 0; ch < HD / 32; ch++) {
                            uint32_t r[32];
                            pr_ld32(my_o + 32 * ch, r);
                            pr_ld32_wait(r);
#pragma unroll
                            for (int x = 0; x < 32; x++) r[x] = __float_as_uint(__uint_as_float(r[x]) * down);
                            pr_st32(my_o + 32 * ch, r);
                        }
                    }
                    m = top;
                    base = top == -INFINITY ? 0.f : top;
                    limit = top + 8.f;
                    l *= down;
                }
                float l0 = 0.f, l1 = 0.f;
#pragma unroll
                for (int ch = 0; ch < 4; ch++) {
                    uint32_t r[32], w[16];
                    pr_ld32(my_s + 32 * ch, r);
                    pr_ld32_wait(r);
                    if (edge) hide(r, ch);
#pragma unroll
                    for (int x = 0; x < 32; x += 2) {
                        const float e0 = exp2_fast(fmaf(__uint_as_float(r[x]), factor, -base)), e1 = exp2_fast(fmaf(__uint_as_float(r[x + 1]), factor, -base));
                        l0 += e0; l1 += e1;
                        w[x / 2] = as_u(__floats2half2_rn(e0, e1));
                    }
                    pr_st16(my_s + 16 * ch, w);
                }
                l += l0 + l1;
                pr_st_wait();
                pr_fence_before();
                __syncwarp();
                if (lane == 0) pr_arrive(smem_at(&p_full[half]));
            }
            pr_wait(smem_at(&o_full[half]), (uint32_t) ((n_s - 1) & 1), dead);
            __syncwarp();
            pr_fence_after();
            const bool final = g.t0 == 0 && g.t1 == g.sp.n;
            const float inv = l != 0.f ? 1.f / l : 0.f;
            const size_t slot = (2 * (size_t) blockIdx.x + (g.t0 == 0 ? 1 : 0)) * PR_COLS + half * 128 + row;
#pragma unroll
            for (int ch = 0; ch < HD / 32; ch++) {
                uint32_t r[32];
                pr_ld32(my_o + 32 * ch, r);
                pr_ld32_wait(r);
                if (in && !dead) {
                    if (final) {
                        T * y = static_cast<T *>(a.out) + ((size_t) (g.q.begin + i) * c.n_kv * a.group + h) * HD + 32 * ch;
#pragma unroll
                        for (int x = 0; x < 32; x += 8) {
                            Eight<T> f;
#pragma unroll
                            for (int j = 0; j < 8; j++) f.v[j] = from_f<T>(__uint_as_float(r[x + j]) * inv);
                            *reinterpret_cast<Eight<T> *>(y + x) = f;
                        }
                    } else {
                        uint4 * y = reinterpret_cast<uint4 *>(a.part + slot * HD + 32 * ch);
#pragma unroll
                        for (int x = 0; x < 8; x++) y[x] = make_uint4(r[4 * x], r[4 * x + 1], r[4 * x + 2], r[4 * x + 3]);
                    }
                }
                __syncwarp();
            }
            if (in && !final) *reinterpret_cast<float2 *>(a.ml + slot * 2) = make_float2(m, l);
            pr_fence_before();
        }
    } else if (warp < 12) {
        const int w = warp - 8, g8 = lane >> 2, tq = lane & 3, tc = g8 >> 1, te = g8 & 1;
        int n = 0;                                                         // tiles so far
        for (long long at = begin; at < end;) {
            const Segment g = segment(at);
            if (!g.run) continue;
            int pages_from = 0, my_page = 0, turned = -1;
            uint4 kr[2][NB / 2], vr[2][NB / 2], ks[2], vs[2][NB / 2];
            const auto place = [&](int t, int u) -> const uint8_t * {      // of 16 tokens
                const int pos = (g.sp.lo + t) * PR_KV + 32 * w + 16 * u, pi = pos >> c.page_log2;
                if (turned < 0 || pi - pages_from >= 32) { turned = 0; pages_from = pi; my_page = page_at(c, g.q.slot, (pi + lane) << c.page_log2); }
                const int page = __shfl_sync(0xffffffffu, my_page, pi - pages_from);
                return page >= 0 ? c.pool + tile_offset(c, page, g.head, pos, TILE) : nullptr;
            };
            const auto ask_k = [&](const uint8_t * const (&src)[2]) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint4 none = make_uint4(0, 0, 0, 0);
                    if constexpr (NB == 4) {
#pragma unroll
                        for (int j = 0; j < 2; j++) kr[u][j] = src[u] ? reinterpret_cast<const uint4 *>(src[u])[32 * j + lane] : none;
                        ks[u] = src[u] ? reinterpret_cast<const uint4 *>(src[u] + 16 * HD)[g8] : none;
                    } else {
                        const uint2 x = src[u] ? reinterpret_cast<const uint2 *>(src[u])[lane] : make_uint2(0, 0), y = src[u] ? reinterpret_cast<const uint2 *>(src[u])[32 + lane] : make_uint2(0, 0);
                        kr[u][0] = make_uint4(x.x, x.y, y.x, y.y);
                        const uint2 z = src[u] ? reinterpret_cast<const uint2 *>(src[u] + 16 * HD)[g8] : make_uint2(0, 0);
                        ks[u] = make_uint4(z.x, z.y, 0, 0);
                    }
                }
            };
            const auto ask_v = [&](const uint8_t * const (&src)[2]) {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < NB / 2; j++) {
                        const uint4 none = make_uint4(0, 0, 0, 0);
                        vr[u][j] = src[u] ? reinterpret_cast<const uint4 *>(src[u] + 8 * HD)[32 * j + lane] : none;
                        vs[u][j] = src[u] ? reinterpret_cast<const uint4 *>(src[u] + 17 * HD)[NB / 2 * tq + j] : none;
                    }
            };
            const uint8_t * src[2] = {place(g.t0, 0), place(g.t0, 1)};
            ask_k(src);
            ask_v(src);
            for (int t = g.t0; t < g.t1; t++, n++) {
                const int stage = n & 1;
                const uint32_t round = (uint32_t) (n >> 1);
                if (t + 1 < g.t1) { src[0] = place(t + 1, 0); src[1] = place(t + 1, 1); }
                if (n >= 2) pr_wait(smem_at(&k_empty[stage]), (round - 1) & 1, dead);
                __syncwarp();
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int row = 32 * w + 8 * tc + 4 * u + 2 * j + te;
#pragma unroll
                        for (int b = 0; b < NB; b++) {
                            const uint4 x = NB == 4 ? kr[u][j & (NB / 2 - 1)] : kr[u][0];
                            const uint32_t word = NB == 4 ? (b == 0 ? x.x : b == 1 ? x.y : b == 2 ? x.z : x.w) : (2 * j + b == 0 ? x.x : 2 * j + b == 1 ? x.y : 2 * j + b == 2 ? x.z : x.w);
                            const int sw = NB == 4 ? 2 * j + b / 2 : j;
                            const __half2 sc = as_h2(sw == 0 ? ks[u].x : sw == 1 ? ks[u].y : sw == 2 ? ks[u].z : ks[u].w), d = b & 1 ? __high2half2(sc) : __low2half2(sc);
                            uint32_t v[4];
                            codes8(word, v);
#pragma unroll
                            for (int x4 = 0; x4 < 4; x4++) v[x4] = as_u(__hmul2(as_h2(v[x4]), d));
                            pr_st_shared(k_s + stage * KVB + (b >> 1) * SUB + row * 128 + (((4 * (b & 1) + tq) ^ (row & 7)) << 4), v[0], v[1], v[2], v[3]);
                        }
                    }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) pr_arrive(smem_at(&k_full[stage]));
                if (t + 1 < g.t1) ask_k(src);
                if (n >= 2) pr_wait(smem_at(&v_empty[stage]), (round - 1) & 1, dead);
                __syncwarp();
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint32_t v[2][2][4];
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const uint4 x = vr[u][b >> 1], z = vs[u][b >> 1];
                            const uint32_t word = b & 1 ? (e ? x.w : x.z) : (e ? x.y : x.x);
                            const __half2 d = as_h2(b & 1 ? (e ? z.w : z.z) : (e ? z.y : z.x));
                            codes8(word, v[u][e]);
#pragma unroll
                            for (int x4 = 0; x4 < 4; x4++) v[u][e][x4] = as_u(__hmul2(as_h2(v[u][e][x4]), d));
                        }
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const int row = 32 * b + 4 * g8 + x;
                        pr_st_shared(v_s + stage * KVB + (w >> 1) * (HD * 128) + row * 128 + (((4 * (w & 1) + tq) ^ (row & 7)) << 4), v[0][0][x], v[0][1][x], v[1][0][x], v[1][1][x]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) pr_arrive(smem_at(&v_full[stage]));
                if (t + 1 < g.t1) ask_v(src);
            }
        }
    } else {
        int n = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
        for (long long at = begin; at < end;) {
            const Segment g = segment(at);
            if (!g.run) continue;
            if (pr_elect()) {
                const int tiles = g.t1 - g.t0;
                const auto scores = [&](int half, int stage) {             // S = Q K^T of a half
#pragma unroll
                    for (int k = 0; k < HD / 16; k++)
                        pr_mma_ss(t_s + half * 128, PR_DESC | (uint64_t) ((q_s + half * QB + (k >> 2) * SUB) >> 4) + 2 * (k & 3), PR_DESC | (uint64_t) ((k_s + stage * KVB + (k >> 2) * SUB) >> 4) + 2 * (k & 3),
                                  pr_idesc(128), k > 0);
                    pr_commit(smem_at(&s_full[half]));
                };
                for (int half = 0; half < g.halves; half++) pr_wait(smem_at(&q_full[half]), (uint32_t) (n_q[half] & 1), dead);
                pr_wait(smem_at(&k_full[n & 1]), (uint32_t) (n >> 1 & 1), dead);
                pr_fence_after();
                if (!dead) {
                    for (int half = 0; half < g.halves; half++) scores(half, n & 1);
                    pr_commit(smem_at(&k_empty[n & 1]));
                }
                for (int t = 0; t < tiles; t++) {
                    const int now = n + t, stage = now & 1, after = (now + 1) & 1;
                    pr_wait(smem_at(&v_full[stage]), (uint32_t) (now >> 1 & 1), dead);
                    for (int half = 0; half < g.halves; half++) {
                        pr_wait(smem_at(&p_full[half]), (uint32_t) ((n_p[half] + t) & 1), dead);
                        pr_fence_after();
                        if (!dead) {
#pragma unroll
                            for (int k = 0; k < PR_KV / 16; k++)
                                pr_mma_ts(t_o + half * HD, t_s + half * 128 + 8 * k, PR_DESC | (uint64_t) ((v_s + stage * KVB + (k >> 2) * (HD * 128)) >> 4) + 2 * (k & 3), pr_idesc(HD), t > 0 || k > 0);
                            pr_commit(smem_at(&o_full[half]));
                        }
                        if (t + 1 < tiles) {
                            if (half == 0) { pr_wait(smem_at(&k_full[after]), (uint32_t) ((now + 1) >> 1 & 1), dead); pr_fence_after(); }
                            if (!dead) {
                                scores(half, after);
                                if (half == g.halves - 1) pr_commit(smem_at(&k_empty[after]));
                            }
                        }
                    }
                    if (!dead) pr_commit(smem_at(&v_empty[stage]));
                }
            }
            __syncwarp();
            n += g.t1 - g.t0;
            for (int half = 0; half < g.halves; half++) { n_q[half]++; n_p[half] += g.t1 - g.t0; }
        }
    }
    if (dead) {
        atomicExch_system(p.err, 1);
        for (int j = 0; j < 1000; j++) __nanosleep(1000);      // products under way end before shared and tensor memory are given back
    }
    pr_fence_before();
    __syncthreads();
    if (warp == 12) {
        pr_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem));
    }
}

// a warp a row and head: adds the parts of a unit that blocks shared, few as they are
template <int HD, typename T>
__global__ void __launch_bounds__(256) k_kv4_prompt_join(const PromptArgs p) {
    constexpr int E = HD / 32;
    const AttendArgs & a = p.a;
    const Cache & c = a.c;
    const int lane = threadIdx.x & 31, n_head = c.n_kv * a.group;
    const int64_t item = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= (int64_t) c.n_rows * n_head) return;
    const int row = (int) (item / n_head), h = (int) (item % n_head), s = seq_of_row(c, row);
    if (s < 0) return;
    const int begin = min(max(c.first[s], 0), c.n_rows), head = h / a.group, col = (row - begin) * a.group + h - head * a.group, ct = col / PR_COLS, in_tile = col - ct * PR_COLS;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int e = p.entry_of[s] + ct, per = p.n_entries[1];
    const long long b0 = a.before[e];
    const int len = (int) ((a.before[e + 1] - b0) / c.n_kv);
    const long long u0 = b0 + (long long) head * len;
    const int w0 = (int) quotient(u0 + PR_OVER, per), w1 = (int) quotient(u0 + len - 1, per);
    if (w0 == w1) return;
    float m = -INFINITY, l = 0.f, o[E] = {};
    for (int w = w0; w <= w1; w++) {
        const size_t slot = (2 * (size_t) w + (w == w0 ? 1 : 0)) * PR_COLS + in_tile;
        const float2 ml = *reinterpret_cast<const float2 *>(a.ml + slot * 2);
        const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.f : top, old = exp2_fast(m - base), now = exp2_fast(ml.x - base);
        l = l * old + ml.y * now;
#pragma unroll
        for (int x = 0; x < E; x++) o[x] = o[x] * old + a.part[slot * HD + E * lane + x] * now;
        m = top;
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    T * y = static_cast<T *>(a.out) + ((size_t) row * n_head + h) * HD + E * lane;
#pragma unroll
    for (int x = 0; x < E; x++) y[x] = from_f<T>(o[x] * inv);
}

}  // namespace srv
}  // namespace b200
