// serve_prompt.cuh — attention of prompts' portions over the 4-bit cache (sm_100a, tcgen05): many rows of a sequence.
//
// A unit of work is 256 columns of a sequence (a column is a row and a query head of one KV head) over the tiles of 128 tokens that they see. As for few rows, all units stand in one
// line that is cut evenly, here over one block per SM; k_kv4_prompt_plan lays the line out, k_kv4_prompt_join adds the parts of units that blocks shared.
//   warps 0-3, 4-7   soft-max of columns 0-127 and 128-255, a thread a column, 64 tokens at a time: its row of S into registers, maximum, exponentials, P back into tensor memory in the
//                    place of S
//   warps 8-11       codes of 32 tokens each, copied ahead, to fp16 in shared memory (exact: a scale has 8 bits, a code 4), K by rows of tokens, V by rows of dims, both with 128-byte swizzle
//   warps 12, 13     (of 12-15: registers are shared out by four warps, 128 a thread at launch, then 168, 168, 112 and 64) one thread each issues a half's S = Q K^T (128 x 64 x head_dim)
//                    and O += P V (P from tensor memory, 128 x head_dim x 64): a thread issues a product every 44 clocks or so, 24 of them a half and tile
// Measured with 32 query heads on 8 of 128: 8192 tokens 552 us (996 TFLOP/s, 59 % of the bf16 rate), 512 rows behind 6000 positions 70 us, of which 5 the plan and 4 the join. What bounds
// it is the chain from S over the soft-max to P: 1750 clocks for 64 tokens, of which 1024 are exponentials (16 a clock), while products read 128 KB of shared memory and codes write 32.
// Sixteen soft-max warps, exponentials in part by polynomials, K made a tile ahead of V and other shares of registers were no faster; one issuing thread 595 us, one turn of 128 tokens 4 % more.
// Tensor memory: S and P [2 halves][2 turns][64 columns], O [2][head_dim]. Each half has two turns of S, so that the scores of the next 64 tokens are there when those in hand are done with.
// Tokens of 32 stand as n = 8 c + 4 u + i for token 16 u + c + 4 i in S, P, K and V alike, and dims of 8 as 0 4 1 5 2 6 3 7 in Q and K: the orders in which a word's codes come apart.
// P is rounded to fp16 (2^-11; P_LIFT and P_PASS in serve_attn.cuh say what that leaves out), q scaled by a power of two into fp16's range; sums are fp32. O is scaled in tensor memory where the
// base of P moves.
// Every wait on an mbarrier is bounded: where one runs out the block raises *err, waits for nothing more, lets what is under way end and frees its tensor memory; the call's results are worthless.
#pragma once
#include "serve_attn.cuh"
#include "../../include/booster_b200.h"
#include <type_traits>

namespace b200 {
namespace srv {

struct Entry { int slot, begin, count, held, ct, lo, n, head; };        // a sequence (Seq), its columns' number, their span of tiles (head: serve_kv16.cuh)
struct PromptArgs {
    AttendArgs a;                        // a.before: [entries + 1] tiles in front of each entry (a sequence's 256 columns), for all KV heads together
    int max_entries;                     // as many as rows and sequences can have, where first ascends; no more are looked at
    Entry * entries;
    int * first;                         // tiles of a block's piece, entries, the entry that each block's piece begins in
    int * err;
    uint32_t polls;                      // of a wait that is given up
    int queries;                         // arrivals that tell a half's queries there (4, one from each warp; 1 of a box in serve_kv16_prompt.cuh), or more than come (b200_kv4_drill)
};

constexpr uint32_t PR_POLLS = 1u << 18;       // a poll that finds nothing takes 7800 clocks: a second
constexpr int PR_COLS = 256, PR_KV = 128, PR_THREADS = 512, PR_OVER = 4;      // PR_OVER: what beginning a unit costs, in tiles (8192 tokens 780 us with 2, 655, 600, 600, 611 with 3, 4, 5, 8)
constexpr uint64_t PR_DESC = (1ull << 16) | ((uint64_t) (1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);      // K-major, 128-byte swizzle, groups of 8 rows 1024 bytes apart
__host__ __device__ constexpr uint32_t pr_idesc(int n) { return (1u << 4) | ((uint32_t) (n >> 3) << 17) | (8u << 24); }     // D f32, A and B f16, M = 128
template <int HD> struct PromptSmem {
    static constexpr int Q = 128 * HD * 2, KV = PR_KV * HD * 2;      // bytes of one half of Q, of a tile's K or V
    static constexpr int BYTES = 2 * Q + 4 * KV + 4 * 36 * HD + 1024;      // K and V in two stages each, a tile's codes as they come
};

__device__ __forceinline__ void pr_wait(uint32_t bar, uint32_t parity, uint32_t polls, bool & dead) {
    for (uint32_t spins = 0; !dead; spins++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) break;
        if (spins >= polls) dead = true;
    }
}
__device__ __forceinline__ void pr_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory"); }
__device__ __forceinline__ void pr_commit(uint32_t bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory"); }
__device__ __forceinline__ void pr_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pr_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
template <int N> __device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N> __device__ __forceinline__ void regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }
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
// 32 columns of a warp's lanes, there when the statement ends: nothing can be put between the load and the wait for it
__device__ __forceinline__ void pr_ld32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(at) : "memory");
}
__device__ __forceinline__ void pr_st32(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
                 :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                    "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
                    "r"(r[30]), "r"(r[31]), "r"(at) : "memory");
}
__device__ __forceinline__ void pr_ld64(uint32_t at, uint32_t (&r)[64]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]) : "r"(at) : "memory");
}
__device__ __forceinline__ void pr_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pr_st_shared(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

__device__ __forceinline__ uint64_t two(float x, float y) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ float2 split(uint64_t p) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p)); return r; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// tiles of 128 tokens that the columns of an entry see, one at least
__device__ __forceinline__ Span prompt_span(const Cache & c, const Seq & q, int group, int window, int ct) {
    const int a = ct * PR_COLS / group, b = min(q.count - 1, (ct * PR_COLS + PR_COLS - 1) / group);
    const int last = min(q.held + b, (c.max_pages << c.page_log2) - 1), first = window > 0 ? max(0, q.held + a - window + 1) : 0;
    Span s;
    s.lo = first / PR_KV;
    s.n = q.slot < 0 || last < first ? 1 : last / PR_KV - s.lo + 1;
    return s;
}

// sum over the threads in front of this one and of the block, of 1024 threads
template <typename V> __device__ __forceinline__ V plan_before(V mine, V & all, V * sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V up = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const V x = __shfl_up_sync(0xffffffffu, up, d); if (lane >= d) up += x; }
    __syncthreads();
    if (lane == 31) sums[warp] = up;
    __syncthreads();
    V part = sums[lane], off = up - mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const V x = __shfl_up_sync(0xffffffffu, part, d); if (lane >= d) part += x; }
    all = __shfl_sync(0xffffffffu, part, 31);
    const V front = __shfl_sync(0xffffffffu, part, (warp + 31) & 31);
    return off + (warp ? front : 0);
}

// one block: the line of entries, a thread an entry. 5 us, its launch and three dependent reads
static __global__ void __launch_bounds__(1024) k_kv4_prompt_plan(const PromptArgs p, int n_blocks) {
    extern __shared__ int entry_of[];                              // [n_seq + 1]
    __shared__ long long sums[32];
    const Cache & c = p.a.c;
    const int tid = threadIdx.x;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int all = 0;
    for (int s0 = 0; s0 < c.n_seq; s0 += 1024) {
        const int s = s0 + tid;
        long long some;
        const long long n = s < c.n_seq ? col_tiles(seq_at(c, s), p.a.group, PR_COLS) : 0, at = all + plan_before(n, some, sums);
        if (s < c.n_seq) entry_of[s] = (int) min(at, (long long) p.max_entries);
        all = (int) min(all + some, (long long) p.max_entries);
    }
    if (tid == 0) entry_of[c.n_seq] = all;
    __syncthreads();
    long long total = 0;
    for (int e0 = 0; e0 < all; e0 += 1024) {
        const int e = e0 + tid;
        long long n = 0, some;
        if (e < all) {
            int s = 0;                                             // the last sequence that begins at or before e (those without rows begin where the next one does)
            for (int hi = c.n_seq; hi - s > 1;) { const int mid = (s + hi) >> 1; if (entry_of[mid] <= e) s = mid; else hi = mid; }
            const Seq q = seq_at(c, s);
            const int ct = e - entry_of[s];
            const Span sp = prompt_span(c, q, p.a.group, p.a.window, ct);
            p.entries[e] = Entry{q.slot, q.begin, q.count, q.held, ct, sp.lo, sp.n, 0};
            n = (long long) c.n_kv * (sp.n + PR_OVER);
        }
        const long long at = total + plan_before(n, some, sums);
        if (e < all) p.a.before[e] = at;
        total += some;
    }
    const int per = (int) max(1ll, quotient(total + n_blocks - 1, n_blocks));
    if (tid == 0) { p.a.before[all] = total; p.first[0] = per; p.first[1] = all; }
    __syncthreads();                                               // before[] stands
    for (int w = tid; w < n_blocks; w += 1024) {                   // the entry that each block's piece begins in
        const long long at = (long long) w * per;
        int e = 0;
        for (int hi = all; hi - e > 1;) { const int mid = (e + hi) >> 1; if (p.a.before[mid] <= at) e = mid; else hi = mid; }
        p.first[2 + w] = e;
    }
}

template <typename T> __device__ __noinline__ uint4 eight_apart(const T * src) {         // where they do not stand on 16 bytes
    const uint16_t * x = reinterpret_cast<const uint16_t *>(src);
    return make_uint4(x[0] | (uint32_t) x[1] << 16, x[2] | (uint32_t) x[3] << 16, x[4] | (uint32_t) x[5] << 16, x[6] | (uint32_t) x[7] << 16);
}
template <typename T> __device__ __forceinline__ float query_entry(const uint4 & f, int j) {    // j: a constant
    const uint32_t w = j >> 1 == 0 ? f.x : j >> 1 == 1 ? f.y : j >> 1 == 2 ? f.z : f.w;
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short) (w >> 16 * (j & 1))));
    else return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
}

// a piece of one unit
struct Segment { Seq q; Span sp; int ct, head, t0, t1, halves; };

// P's columns hold tokens in this order (of 32)
__host__ __device__ constexpr int token_of(int col) { return 16 * (col >> 2 & 1) + (col >> 3) + 4 * (col & 3); }

template <int HD, typename T>
__global__ void __launch_bounds__(PR_THREADS, 1) k_kv4_prompt(const PromptArgs p) {
    constexpr int NB = HD / 32, TILE = 18 * HD, QB = PromptSmem<HD>::Q, KVB = PromptSmem<HD>::KV, SUB = 128 * 128;      // SUB: 128 rows of 128 bytes
    extern __shared__ uint8_t pr_raw[];
    __shared__ __align__(8) uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], o_full[2][2];      // [half][turn]
    __shared__ uint32_t tmem_s;
    const AttendArgs & a = p.a;
    const Cache & c = a.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t smem = (smem_at(pr_raw) + 1023u) & ~1023u, q_s = smem, k_s = q_s + 2 * QB, v_s = k_s + 2 * KVB;
    if (tid == 0) {
        const auto init = [](uint64_t * b, int n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(smem_at(b)), "r"(n) : "memory"); };
        for (int i = 0; i < 2; i++) { init(&q_full[i], p.queries); init(&k_full[i], 4); init(&v_full[i], 4); init(&k_empty[i], 2); init(&v_empty[i], 2); for (int b = 0; b < 2; b++) { init(&s_full[i][b], 1); init(&p_full[i][b], 4); init(&o_full[i][b], 1); } }
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
    const int per = p.first[0], entries = p.first[1];
    const long long begin = (long long) blockIdx.x * per, end = min(a.before[entries], begin + per);
    // the segments of this block's piece, one after the other and the same for every warp
    int entry = begin < end ? p.first[2 + blockIdx.x] : 0, head = -1;
    long long at = begin;
    const auto segment = [&](Segment & g) {
        while (at < end) {
            const Entry e = p.entries[entry];
            const int len = e.n + PR_OVER;
            int from = 0;
            if (head < 0) {                                        // the first one may begin anywhere
                const long long x = at - a.before[entry];
                head = (int) quotient(x, len);
                from = (int) (x - (long long) head * len);
            }
            const int to = (int) min((long long) len, from + (end - at));
            g.q = Seq{e.slot, e.begin, e.count, e.held};
            g.sp = Span{e.lo, e.n};
            g.ct = e.ct; g.head = head;
            g.t0 = max(0, from - PR_OVER);
            g.t1 = to - PR_OVER;
            g.halves = e.count * a.group - e.ct * PR_COLS > 128 ? 2 : 1;
            at += to - from;
            if (++head == c.n_kv) { head = 0; entry++; }
            if (g.t1 > 0) return true;
        }
        return false;
    };
    bool dead = false;
    if (warp < 8) {
        regs_more<168>();
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;          // of the half
        const uint32_t lanes = (uint32_t) ((warp & 3) * 32) << 16, my_s = t_s + lanes + half * 128, my_o = t_o + lanes + half * HD;
        int n_s = 0;                                                       // steps of 64 tokens of this half so far
        const auto next = [&](Segment & g) {                               // the next segment with columns of this half
            do { if (!segment(g)) return false; } while (half >= g.halves);
            return true;
        };
        // the warp's 32 queries, HD / 8 lanes a row: each scaled by a power of two to at most 2^14, dims of eight as 0 4 1 5 2 6 3 7. Returns what the column's scores are scaled by
        const auto queries = [&](const Segment & g) {
            const int col = g.ct * PR_COLS + half * 128 + row, i = col / a.group, h = g.head * a.group + col - i * a.group;
            const bool in = i < g.q.count;
            constexpr int LANES = HD / 8, ROWS = 32 / LANES, X = 8;
            float factor = 0.f;
            {
                const int64_t mine = in ? (g.q.begin + i) * a.q_row + h * a.q_head : -1;
                const int m = lane % LANES;
#pragma unroll 1
                for (int x0 = 0; x0 < 32; x0 += X * ROWS) {
                    uint4 f[X];
                    int64_t from[X];
#pragma unroll
                    for (int x = 0; x < X; x++) { from[x] = __shfl_sync(0xffffffffu, mine, x0 + x * ROWS + lane / LANES); f[x] = make_uint4(0, 0, 0, 0); }
                    const T * src = static_cast<const T *>(a.q) + 8 * m;
                    if (a.q_whole) {
#pragma unroll
                        for (int x = 0; x < X; x++) if (from[x] >= 0) f[x] = *reinterpret_cast<const uint4 *>(src + from[x]);
                    } else {
#pragma unroll
                        for (int x = 0; x < X; x++) if (from[x] >= 0) f[x] = eight_apart(src + from[x]);
                    }
#pragma unroll
                    for (int x = 0; x < X; x++) {
                        const int r = x0 + x * ROWS + lane / LANES;
                        float top = 0.f;
#pragma unroll
                        for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(query_entry<T>(f[x], j)));
#pragma unroll
                        for (int d = 1; d < LANES; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        float up = query_scale(top);
                        const float mine_up = __shfl_sync(0xffffffffu, up, (lane % ROWS) * LANES);
                        if (lane / ROWS == x0 / ROWS + x) factor = mine_up;
                        if (a.scale_log2 < 0.f) up = -up;
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; j++) w[j] = as_u(__floats2half2_rn(query_entry<T>(f[x], j) * up, query_entry<T>(f[x], j + 4) * up));
                        pr_st_shared(q_s + half * QB + (m >> 3) * SUB + ((warp & 3) * 32 + r) * 128 + (((m & 7) ^ (r & 7)) << 4), w[0], w[1], w[2], w[3]);
                    }
                }
                factor = fmaxf(fabsf(a.scale_log2) / factor, 1.2e-38f);              // (never 0: it meets the -infinity of what is masked)
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) pr_arrive(smem_at(&q_full[half]));
            return factor;
        };
        Segment g;
        bool more = next(g);
        float factor = more ? queries(g) : 0.f;
        while (more) {
            const int col = g.ct * PR_COLS + half * 128 + row, i = col / a.group, h = g.head * a.group + col - i * a.group;
            const bool in = i < g.q.count;
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
            for (int t = 2 * g.t0; t < 2 * g.t1; t++, n_s++) {
                const int pos = g.sp.lo * PR_KV + 64 * t;
                const uint32_t at = my_s + 64 * (n_s & 1);
                const bool edge = !whole || pos + 63 > all_see_hi || pos < all_see_lo;
                unsigned there = 0xfu;                                     // tiles of 16 tokens that have a page
                if (!whole) there = __ballot_sync(0xffffffffu, lane < 4 && page_at(c, g.q.slot, pos + 16 * (lane & 3)) >= 0);
                pr_wait(smem_at(&s_full[half][n_s & 1]), (uint32_t) (n_s >> 1 & 1), p.polls, dead);
                __syncwarp();
                pr_fence_after();
                uint32_t r[64];
                pr_ld64(at, r);
                if (edge) {                                                // what a column does not see goes to -infinity
                    const int hi = top_pos - pos, lo = low_pos - pos;
#pragma unroll
                    for (int x = 0; x < 64; x++) {
                        const int token = (x & 32) + token_of(x & 31);
                        if (token > hi || token <= lo || !(there >> (token >> 4) & 1)) r[x] = 0xff800000u;
                    }
                }
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int x = 0; x < 64; x += 4) {
                    x0 = fmaxf(x0, fmaxf(__uint_as_float(r[x]), __uint_as_float(r[x + 1])));
                    x1 = fmaxf(x1, fmaxf(__uint_as_float(r[x + 2]), __uint_as_float(r[x + 3])));
                }
                const float high = fmaxf(x0, x1), score = high == -INFINITY ? high : high * factor;
                if (__any_sync(0xffffffffu, score > limit)) {
                    const float top = fmaxf(m, score - P_LIFT), down = top > m ? exp2_fast(m - top) : 1.f;
                    if (t > 2 * g.t0 && __any_sync(0xffffffffu, down != 1.f)) {
                        pr_wait(smem_at(&o_full[half][(n_s - 1) & 1]), (uint32_t) ((n_s - 1) >> 1 & 1), p.polls, dead);
                        __syncwarp();
                        pr_fence_after();
#pragma unroll 1
                        for (int ch = 0; ch < HD / 32; ch++) {
                            uint32_t y[32];
                            pr_ld32(my_o + 32 * ch, y);
#pragma unroll
                            for (int x = 0; x < 32; x++) y[x] = __float_as_uint(__uint_as_float(y[x]) * down);
                            pr_st32(my_o + 32 * ch, y);
                        }
                    }
                    m = top;
                    base = top == -INFINITY ? 0.f : top;
                    limit = top + (P_LIFT + P_PASS);
                    l *= down;
                }
                const uint64_t by = two(factor, factor), less = two(-base, -base);
                uint64_t sum = 0;
                uint32_t w[32];
#pragma unroll
                for (int x = 0; x < 64; x += 2) {
                    const float2 y = split(fma2(two(__uint_as_float(r[x]), __uint_as_float(r[x + 1])), by, less));
                    const float e0 = exp2_fast(y.x), e1 = exp2_fast(y.y);
                    sum = add2(sum, two(e0, e1));
                    w[x / 2] = as_u(__floats2half2_rn(e0, e1));
                }
                pr_st32(at, w);
                l += split(sum).x + split(sum).y;
                pr_st_wait();
                pr_fence_before();
                __syncwarp();
                if (lane == 0) pr_arrive(smem_at(&p_full[half][n_s & 1]));
            }
            // the next segment's queries before this one's results: its first scores are made while these are written
            Segment then;
            more = next(then);
            if (more) factor = queries(then);
            pr_wait(smem_at(&o_full[half][(n_s - 1) & 1]), (uint32_t) ((n_s - 1) >> 1 & 1), p.polls, dead);
            __syncwarp();
            pr_fence_after();
            const bool final = g.t0 == 0 && g.t1 == g.sp.n;
            const float inv = l != 0.f ? 1.f / l : 0.f;
            const size_t piece = 2 * (size_t) blockIdx.x + (g.t0 == 0 ? 1 : 0);      // parts are [HD / 4][256 columns][4]: a warp's stores are contiguous
#pragma unroll
            for (int ch = 0; ch < HD / 32; ch++) {
                uint32_t r[32];
                pr_ld32(my_o + 32 * ch, r);
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
                        uint4 * y = reinterpret_cast<uint4 *>(a.part + piece * PR_COLS * HD) + (size_t) (8 * ch) * PR_COLS + half * 128 + row;
#pragma unroll
                        for (int x = 0; x < 8; x++) y[x * PR_COLS] = make_uint4(r[4 * x], r[4 * x + 1], r[4 * x + 2], r[4 * x + 3]);
                    }
                }
                __syncwarp();
            }
            if (in && !final) *reinterpret_cast<float2 *>(a.ml + (piece * PR_COLS + half * 128 + row) * 2) = make_float2(m, l);
            pr_fence_before();
            g = then;
        }
    } else if (warp < 12) {
        regs_less<112>();
        const int w = warp - 8, g8 = lane >> 2, tq = lane & 3, tc = g8 >> 1, te = g8 & 1;
        int n = 0;                                                         // tiles so far
        const uint32_t raw_s = v_s + 2 * KVB + (uint32_t) (w * 2 * TILE);
        const uint8_t * raw = pr_raw + (raw_s - smem_at(pr_raw));
        for (Segment g; segment(g);) {
            int pages_from = 0, my_page = 0;
            bool turned = false;
            const auto page_of = [&](int pos) {
                const int pi = pos >> c.page_log2;
                if (!turned || pi - pages_from >= 32) { turned = true; pages_from = pi; my_page = page_at(c, g.q.slot, (pi + lane) << c.page_log2); }
                return __shfl_sync(0xffffffffu, my_page, pi - pages_from);
            };
            const auto ask = [&](int t) {                                  // the warp's 32 tokens, zeros where there is no page
                const int pos = (g.sp.lo + t) * PR_KV + 32 * w, page_a = page_of(pos), page_b = page_of(pos + 16);
                PairSrc src;
                src.bytes_a = page_a >= 0 ? 16 : 0;
                src.bytes_b = page_b >= 0 ? 16 : 0;
                src.a = c.pool + (page_a >= 0 ? tile_offset(c, page_a, g.head, pos, TILE) : 0) + 16 * lane;
                src.b = c.pool + (page_b >= 0 ? tile_offset(c, page_b, g.head, pos + 16, TILE) - TILE : 0) + 16 * lane;
                const bool first = lane < TILE % 512 / 16;
                src.mid = first ? src.a : src.b; src.bytes_mid = first ? src.bytes_a : src.bytes_b;
                copy_pair<HD>(raw_s + 16 * lane, src, lane);
            };
            ask(g.t0);
            for (int t = g.t0; t < g.t1; t++, n++) {
                const int stage = n & 1;
                const uint32_t round = (uint32_t) (n >> 1);
                asm volatile("cp.async.wait_all;" ::: "memory");
                if (n >= 2) pr_wait(smem_at(&k_empty[stage]), (round - 1) & 1, p.polls, dead);
                __syncwarp();
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint8_t * tile = raw + u * TILE;
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const int row = 32 * w + 8 * tc + 4 * u + 2 * j + te;
                        uint32_t words[NB], scales[NB / 2];
                        if constexpr (NB == 4) {
                            const uint4 x = reinterpret_cast<const uint4 *>(tile)[32 * j + lane];
                            const uint2 z = reinterpret_cast<const uint2 *>(tile + 16 * HD)[2 * g8 + j];
                            words[0] = x.x; words[1] = x.y; words[2] = x.z; words[3] = x.w; scales[0] = z.x; scales[1] = z.y;
                        } else {
                            const uint2 x = reinterpret_cast<const uint2 *>(tile)[32 * j + lane];
                            words[0] = x.x; words[1] = x.y; scales[0] = reinterpret_cast<const uint32_t *>(tile + 16 * HD)[2 * g8 + j];
                        }
#pragma unroll
                        for (int b = 0; b < NB; b++) {
                            const __half2 sc = as_h2(scales[b >> 1]), d = b & 1 ? __high2half2(sc) : __low2half2(sc);
                            uint32_t v[4];
                            codes8(words[b], v);
#pragma unroll
                            for (int x4 = 0; x4 < 4; x4++) v[x4] = as_u(__hmul2(as_h2(v[x4]), d));
                            pr_st_shared(k_s + stage * KVB + (b >> 1) * SUB + row * 128 + (((4 * (b & 1) + tq) ^ (row & 7)) << 4), v[0], v[1], v[2], v[3]);
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) pr_arrive(smem_at(&k_full[stage]));
                if (n >= 2) pr_wait(smem_at(&v_empty[stage]), (round - 1) & 1, p.polls, dead);
                __syncwarp();
#pragma unroll
                for (int bb = 0; bb < NB / 2; bb++) {
                    uint4 y[2], z[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) { y[u] = reinterpret_cast<const uint4 *>(raw + u * TILE + 8 * HD)[32 * bb + lane]; z[u] = reinterpret_cast<const uint4 *>(raw + u * TILE + 17 * HD)[NB / 2 * tq + bb]; }
#pragma unroll
                    for (int b = 2 * bb; b < 2 * bb + 2; b++) {
                        uint32_t v[2][2][4];
#pragma unroll
                        for (int u = 0; u < 2; u++)
#pragma unroll
                            for (int e = 0; e < 2; e++) {
                                codes8(b & 1 ? (e ? y[u].w : y[u].z) : (e ? y[u].y : y[u].x), v[u][e]);
                                const __half2 d = as_h2(b & 1 ? (e ? z[u].w : z[u].z) : (e ? z[u].y : z[u].x));
#pragma unroll
                                for (int x4 = 0; x4 < 4; x4++) v[u][e][x4] = as_u(__hmul2(as_h2(v[u][e][x4]), d));
                            }
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const int row = 32 * b + 4 * g8 + x;
                            pr_st_shared(v_s + stage * KVB + (w >> 1) * (HD * 128) + row * 128 + (((4 * (w & 1) + tq) ^ (row & 7)) << 4), v[0][0][x], v[0][1][x], v[1][0][x], v[1][1][x]);
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) pr_arrive(smem_at(&v_full[stage]));
                if (t + 1 < g.t1) ask(t + 1);
            }
        }
        for (int i = max(0, n - 2); i < n; i++) {                          // the last tiles are let go: their commits arrive while the block's shared memory is its own
            pr_wait(smem_at(&k_empty[i & 1]), (uint32_t) (i >> 1 & 1), p.polls, dead);
            pr_wait(smem_at(&v_empty[i & 1]), (uint32_t) (i >> 1 & 1), p.polls, dead);
        }
    } else {
        regs_less<64>();
        const int half = warp - 12;
        int n = 0, n_q = 0, n_p = 0;                                       // tiles, segments and steps of this half so far
        for (Segment g; half < 2 && segment(g);) {
            const int tiles = g.t1 - g.t0, steps = 2 * tiles;
            if (pr_elect()) {
                if (half < g.halves) {
                    const auto scores = [&](int step) {                    // S = Q K^T of 64 tokens
                        const int turn = step & 1;
#pragma unroll
                        for (int k = 0; k < HD / 16; k++)
                            pr_mma_ss(t_s + half * 128 + 64 * turn, PR_DESC | (uint64_t) ((q_s + half * QB + (k >> 2) * SUB) >> 4) + 2 * (k & 3),
                                      PR_DESC | (uint64_t) ((k_s + (n + (step >> 1) & 1) * KVB + (k >> 2) * SUB + turn * (SUB / 2)) >> 4) + 2 * (k & 3), pr_idesc(64), k > 0);
                        pr_commit(smem_at(&s_full[half][turn]));
                    };
                    pr_wait(smem_at(&q_full[half]), (uint32_t) (n_q & 1), p.polls, dead);
                    pr_wait(smem_at(&k_full[n & 1]), (uint32_t) (n >> 1 & 1), p.polls, dead);
                    pr_fence_after();
                    if (!dead) {
                        scores(0);
                        scores(1);
                        pr_commit(smem_at(&k_empty[n & 1]));
                    }
                    for (int step = 0; step < steps; step++) {
                        const int turn = step & 1, now = n + (step >> 1), stage = now & 1, after = (now + 1) & 1;
                        if (turn == 0) pr_wait(smem_at(&v_full[stage]), (uint32_t) (now >> 1 & 1), p.polls, dead);
                        pr_wait(smem_at(&p_full[half][turn]), (uint32_t) ((n_p + step) >> 1 & 1), p.polls, dead);
                        pr_fence_after();
                        if (!dead) {
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                pr_mma_ts(t_o + half * HD, t_s + half * 128 + 64 * turn + 8 * k, PR_DESC | (uint64_t) ((v_s + stage * KVB + turn * (HD * 128)) >> 4) + 2 * k, pr_idesc(HD), step > 0 || k > 0);
                            pr_commit(smem_at(&o_full[half][turn]));
                            if (turn == 1) pr_commit(smem_at(&v_empty[stage]));
                        }
                        if (step + 2 < steps) {
                            if (turn == 0) { pr_wait(smem_at(&k_full[after]), (uint32_t) ((now + 1) >> 1 & 1), p.polls, dead); pr_fence_after(); }
                            if (!dead) {
                                scores(step + 2);
                                if (turn == 1) pr_commit(smem_at(&k_empty[after]));
                            }
                        }
                    }
                } else {                                                   // no columns here: the tiles are let go as they come
                    for (int t = 0; t < tiles; t++) {
                        const int stage = (n + t) & 1;
                        const uint32_t phase = (uint32_t) ((n + t) >> 1 & 1);
                        pr_wait(smem_at(&k_full[stage]), phase, p.polls, dead);
                        if (!dead) pr_arrive(smem_at(&k_empty[stage]));
                        pr_wait(smem_at(&v_full[stage]), phase, p.polls, dead);
                        if (!dead) pr_arrive(smem_at(&v_empty[stage]));
                    }
                }
            }
            __syncwarp();
            n += tiles;
            if (half < g.halves) { n_q++; n_p += steps; }
        }
    }
    if (dead) atomicExch_system(p.err, 1);
    pr_fence_before();
    if (__syncthreads_or(dead))                                            // nobody issues any more: products under way end before shared and tensor memory are given back
        for (int j = 0; j < 1000; j++) __nanosleep(1000);
    if (warp == 12) {
        pr_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem));
    }
}

// a block 32 columns of a unit that blocks shared: adds its parts, few as they are (4 us behind the kernel in front). A lane is a column, a warp has every eighth group of 4 dims
template <int HD, typename T>
__global__ void __launch_bounds__(256) k_kv4_prompt_join(const PromptArgs p) {
    constexpr int X = HD / 32, PAD = HD + 4;
    __shared__ __align__(16) float sums[32 * PAD];
    const AttendArgs & a = p.a;
    const Cache & c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x / (PR_COLS / 32), c0 = blockIdx.x % (PR_COLS / 32) * 32, head = blockIdx.y;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (e >= p.first[1]) return;
    const Entry n = p.entries[e];
    const int len = n.n + PR_OVER, per = p.first[0], cols = min(PR_COLS, n.count * a.group - n.ct * PR_COLS);
    if (c0 >= cols) return;
    const long long u0 = a.before[e] + (long long) head * len;
    const int w0 = (int) quotient(u0 + PR_OVER, per), w1 = (int) quotient(u0 + len - 1, per);
    if (w0 == w1) return;
    float m = -INFINITY, l = 0.f, o[X][4] = {};
    for (int w = w0; w <= w1; w++) {
        const size_t part = 2 * (size_t) w + (w == w0 ? 1 : 0);
        const bool in = c0 + lane < cols;                          // (others were not stored)
        const float2 ml = in ? *reinterpret_cast<const float2 *>(a.ml + (part * PR_COLS + c0 + lane) * 2) : make_float2(-INFINITY, 0.f);
        float4 v[X];
#pragma unroll
        for (int x = 0; x < X; x++) v[x] = in ? reinterpret_cast<const float4 *>(a.part + part * PR_COLS * HD)[(size_t) (warp + 8 * x) * PR_COLS + c0 + lane] : make_float4(0.f, 0.f, 0.f, 0.f);
        const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.f : top, old = exp2_fast(m - base), now = exp2_fast(ml.x - base);
        l = l * old + ml.y * now;
#pragma unroll
        for (int x = 0; x < X; x++) {
            o[x][0] = o[x][0] * old + v[x].x * now; o[x][1] = o[x][1] * old + v[x].y * now;
            o[x][2] = o[x][2] * old + v[x].z * now; o[x][3] = o[x][3] * old + v[x].w * now;
        }
        m = top;
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int x = 0; x < X; x++) *reinterpret_cast<float4 *>(sums + lane * PAD + 4 * (warp + 8 * x)) = make_float4(o[x][0] * inv, o[x][1] * inv, o[x][2] * inv, o[x][3] * inv);
    __syncthreads();
    for (int x = warp; x < 32 && c0 + x < cols; x += 8) {
        const int col = n.ct * PR_COLS + c0 + x, i = col / a.group, h = head * a.group + col - i * a.group;
        T * y = static_cast<T *>(a.out) + ((size_t) (n.begin + i) * c.n_kv * a.group + h) * HD + X * lane;
#pragma unroll
        for (int j = 0; j < X; j++) y[j] = from_f<T>(sums[x * PAD + X * lane + j]);
    }
}

// ---- host: the workspace of a step ----
inline int64_t prompt_entries(const b200_kv4 & c, int group) { return (int64_t) c.n_rows * group / PR_COLS + c.n_seq + 1; }
struct PromptWork { int64_t entries, first, ml, part, bytes; };       // places in the workspace; `before` is first
inline PromptWork prompt_work(const b200_kv4 & c, int group, int sms) {
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

}  // namespace srv
}  // namespace b200
