// serve_kv16_prompt.cuh — attention of many rows of a sequence over the 16-bit cache (sm_100a, tcgen05): prompts' portions, and the drafts of sequences whose heads share keys.
//
// As over the 4-bit cache (serve_prompt.cuh): a unit of work is 256 columns of a sequence (a column is a row and a query head of one KV head) over the tiles of 128 tokens that they see; all units
// stand in one line that is cut evenly over one block per SM, k_kv16_plan lays it out and k_kv16_prompt_join adds the parts of units that blocks shared. Under a window a unit's tiles are those of
// the first tokens and those of the window.
//   warps 0-3, 4-7   soft-max of columns 0-127 and 128-255, a thread a column, 64 tokens at a time: its row of S into registers, maximum, exponentials, P back into tensor memory in the
//                    place of S
//   warp 8           (of 8-11: registers are shared out by four warps, 168 a thread at launch, then 216, 216 and 72) tiles by TMA, a lane a page: K as rows of tokens, V as it stands too, since
//                    the second product takes its B operand with the dims contiguous (MN-major)
//   warps 9, 10      one thread each issues a half's S = Q K^T (128 x 64 x head_dim) and O += P V (P from tensor memory, 128 x head_dim x 64)
//   warp 11          the next segment's queries, while the last 128 tokens of the one before are worked on, where 128 columns are whole rows of a group: a box. Others the soft-max warps gather
// Tensor memory: S and P [2 halves][2 turns][64 columns], O [2][head_dim]. Each half has two turns of S, so that the scores of the next 64 tokens are there when those in hand are done with.
// P is rounded to the type once, with p16_lift of serve_kv16.cuh: results are off by 1.2 to 1.35 times (rms) what their own rounding is (bfloat16 2.1e-3 for 1.7e-3, fp16 2.8e-4 for 2.1e-4).
// In two numbers, as for few rows, the second product would be twice as long; sums of the rounded weights instead of the weights' made 8192 tokens 45 us longer and no result nearer.
// O is scaled in tensor memory where the base of P moves.
// Measured with 32 query heads on 8 of 128: 8192 tokens 467 us (1177 TFLOP/s, 71 % of the bf16 rate; 522 in calls one after another, which the card's power bounds), 1000 rows behind 5000 positions 100 us by
// itself behind other work, 107 in calls from Python on inputs that change, of which 5 the plan and 10 the join. A step of 64
// tokens takes 1750 clocks: of both halves' products 1280 (those of 64 tokens read 6 KB of shared memory in 48 clocks, for 32 of arithmetic), of exponentials 900, an eighth of them by a
// polynomial (none 495 us, two eighths 489, three 494). Halves that took turns at exponentials by named barriers 475 to 485 and nothing at 1000 rows. What a warp does between them bounds it: a wait for
// what is there 130 clocks, 64 scores from tensor memory 60 to 120, the largest 280, P back 120.
// Every wait on an mbarrier is bounded: where one runs out the block raises *err, waits for nothing more, lets what is under way end and frees its tensor memory; the call's results are worthless.
#pragma once
#include "serve_kv16.cuh"
#include "serve_prompt.cuh"

namespace b200 {
namespace srv {

// P16_OVER: what beginning a unit costs, in tiles. With 1, 2, 3, 4, 6, us: 2000 tokens 65, 57, 56, 57, 59; ragged portions 107, 99, 98, 100, 103; 1000 rows behind 5000 90, 90, 90, 91, 93; 48 sequences of 8 rows 88, 89, 90, 92, 95
constexpr int P16_THREADS = 384, P16_OVER = 3;
constexpr int P16_EIGHTHS = 1;
template <typename T> __host__ __device__ constexpr uint32_t p16_idesc(int n, bool b_by_dims) {      // D f32, A and B of T, M = 128
    const uint32_t t = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (t << 7) | (t << 10) | (b_by_dims ? 1u << 16 : 0u) | ((uint32_t) (n >> 3) << 17) | (8u << 24);
}
// V as [64 dims' half][128 tokens][64 dims]: blocks of 64 dims 16384 bytes apart, groups of 8 tokens 1024
constexpr uint64_t P16_V_DESC = ((uint64_t) (16384u >> 4) << 16) | ((uint64_t) (1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
template <int HD> struct Prompt16Smem {
    static constexpr int Q = 128 * HD * 2, KV = PR_KV * HD * 2;      // bytes of one half of Q, of a tile's K or V
    static constexpr int BYTES = 2 * Q + 4 * KV + 1024;              // K and V in two stages each
};
// the box's tokens of 64 dims of a KV head of a page, keys (side 0) or values
__device__ __forceinline__ void tma_side(uint32_t dst, const CUtensorMap * map, uint32_t bar, int dim, int token, int head, int side, int page) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
                 :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(dim), "r"(token), "r"(head), "r"(side), "r"(page) : "memory");
}

// 64 dims of the queries of 128 columns: rows of a head's group one after the other
__device__ __forceinline__ void tma_queries(uint32_t dst, const CUtensorMap * map, uint32_t bar, int dim, int head, int row) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 :: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(dim), "r"(head), "r"(row) : "memory");
}

// 2^y of two numbers without the special functions' unit: y = n + f with |f| <= 1 / 2, a polynomial of the fourth degree that fits 2^f to 2^-18.5 (least largest relative error, by weighted least
// squares on Chebyshev's places), times 2^n made from n's bits. 0 from y = -127 down; a NaN stays one
__device__ __forceinline__ float max_of_nan(float x, float y) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float2 exp2_pair(float2 y) {
    constexpr float WHOLE = 12582912.f;                                  // 1.5 x 2^23: added, the last bits are a whole number
    const uint64_t x = two(max_of_nan(y.x, -127.f), max_of_nan(y.y, -127.f)), t = add2(x, two(WHOLE, WHOLE)), f = fma2(add2(t, two(-WHOLE, -WHOLE)), two(-1.f, -1.f), x);
    uint64_t p = fma2(f, two(0.009570100344717503f, 0.009570100344717503f), two(0.05591785907745361f, 0.05591785907745361f));
    p = fma2(p, f, two(0.240247443318367f, 0.240247443318367f));
    p = fma2(p, f, two(0.6931217908859253f, 0.6931217908859253f));
    p = fma2(p, f, two(0.9999992847442627f, 0.9999992847442627f));
    const float2 n = split(t);
    const auto power = [](float n) { return __uint_as_float((__float_as_uint(n) << 23) + 0x3f800000u); };
    return split(mul2(p, two(power(n.x), power(n.y))));
}
// the lowest n bits
__device__ __forceinline__ uint64_t first_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// one block: the line of entries, a thread an entry
static __global__ void __launch_bounds__(1024) k_kv16_plan(const PromptArgs p, int n_blocks) {
    extern __shared__ int entry_of[];                              // [n_seq + 1]
    __shared__ long long sums[32];
    const Cache & c = p.a.c;
    const int tid = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
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
            const int ct = e - entry_of[s], a = ct * PR_COLS / p.a.group, b = min(q.count - 1, (ct * PR_COLS + PR_COLS - 1) / p.a.group);
            const Steps sp = steps_of(c, q, p.a.window, p.a.sinks, a, b, 7);
            p.entries[e] = Entry{q.slot, q.begin, q.count, q.held, ct, sp.lo, sp.n, sp.head};
            n = (long long) c.n_kv * (sp.n + P16_OVER);
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

struct Segment16 { Seq q; Steps sp; int ct, head, t0, t1, halves, n0; };      // n0: the block's tiles in front of it

template <int HD, typename T>
__global__ void __launch_bounds__(P16_THREADS, 1) k_kv16_prompt(const PromptArgs p, const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap q_map, bool by_box) {
    constexpr int QB = Prompt16Smem<HD>::Q, KVB = Prompt16Smem<HD>::KV, SUB = 128 * 128;      // SUB: 128 rows of 128 bytes
    extern __shared__ uint8_t pr_raw[];
    __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], o_full[2][2];      // [half][turn]
    __shared__ uint32_t tmem_s, there_s[4];                      // there_s: of a tile, its sixteens of tokens that have a page
    const AttendArgs & a = p.a;
    const Cache & c = a.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const uint32_t smem = (smem_at(pr_raw) + 1023u) & ~1023u, q_s = smem, k_s = q_s + 2 * QB, v_s = k_s + 2 * KVB;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(smem_at(&q_full[i]), p.queries); mbar_init(smem_at(&q_empty[i]), 5);
            mbar_init(smem_at(&k_full[i]), 1); mbar_init(smem_at(&v_full[i]), 1);
            mbar_init(smem_at(&k_empty[i]), 2); mbar_init(smem_at(&v_empty[i]), 2);
            for (int b = 0; b < 2; b++) { mbar_init(smem_at(&s_full[i][b]), 1); mbar_init(smem_at(&p_full[i][b]), 4); mbar_init(smem_at(&o_full[i][b]), 1); }
        }
        mbar_init_done();
    }
    if (warp == 8) {
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
    int entry = begin < end ? p.first[2 + blockIdx.x] : 0, head = -1, tiles_before = 0;
    long long at = begin;
    const auto segment = [&](Segment16 & g) {
        while (at < end) {
            const Entry e = p.entries[entry];
            const int len = e.n + P16_OVER;
            int from = 0;
            if (head < 0) {                                        // the first one may begin anywhere
                const long long x = at - a.before[entry];
                head = (int) quotient(x, len);
                from = (int) (x - (long long) head * len);
            }
            const int to = (int) min((long long) len, from + (end - at));
            g.q = Seq{e.slot, e.begin, e.count, e.held};
            g.sp = Steps{e.head, e.lo, e.n};
            g.ct = e.ct; g.head = head;
            g.t0 = max(0, from - P16_OVER);
            g.t1 = to - P16_OVER;
            g.halves = e.count * a.group - e.ct * PR_COLS > 128 ? 2 : 1;
            at += to - from;
            if (++head == c.n_kv) { head = 0; entry++; }
            if (g.t1 > 0) {
                g.n0 = tiles_before;
                tiles_before += g.t1 - g.t0;
                return true;
            }
        }
        return false;
    };
    bool dead = false;
    if (warp < 8) {
        regs_more<216>();
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;          // of the half
        const uint32_t lanes = (uint32_t) ((warp & 3) * 32) << 16, my_s = t_s + lanes + half * 128, my_o = t_o + lanes + half * HD;
        const float factor = fmaxf(fabsf(a.scale_log2), 1.2e-38f);         // (never 0: it meets the -infinity of what is masked)
        const bool turned = a.scale_log2 < 0.f;
        int n_s = 0, n_q = 0;                                              // steps of 64 tokens and segments of this half so far
        const auto next = [&](Segment16 & g) {                             // the next segment with columns of this half
            do { if (!segment(g)) return false; } while (half >= g.halves);
            return true;
        };
        // the warp's 32 queries where boxes do not bring them: HD / 8 lanes a row
        const auto queries = [&](const Segment16 & g) {
            const int col = g.ct * PR_COLS + half * 128 + row, i = col / a.group, h = g.head * a.group + col - i * a.group;
            constexpr int LANES = HD / 8, ROWS = 32 / LANES, X = HD == 128 ? 4 : 8;
            const int64_t mine = i < g.q.count ? (g.q.begin + i) * a.q_row + h * a.q_head : -1;
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
                    pr_st_shared(q_s + half * QB + (m >> 3) * SUB + ((warp & 3) * 32 + r) * 128 + (((m & 7) ^ (r & 7)) << 4), f[x].x, f[x].y, f[x].z, f[x].w);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) pr_arrive(smem_at(&q_full[half]));
        };
        Segment16 g;
        bool more = next(g);
        if (more && !by_box) queries(g);
        while (more) {
            const int col = g.ct * PR_COLS + half * 128 + row, i = col / a.group, h = g.head * a.group + col - i * a.group;
            const bool in = i < g.q.count;
            const int row_lo = g.ct * PR_COLS / a.group, row_hi = min(g.q.count - 1, (g.ct * PR_COLS + PR_COLS - 1) / a.group);
            const int all_see_hi = g.q.held + row_lo, all_see_lo = a.window > 0 ? g.q.held + row_hi - a.window + 1 : 0;
            const int top_pos = in ? g.q.held + i : -1, low_pos = a.window > 0 ? top_pos - a.window : -1;      // sees low_pos < position <= top_pos, and what is below sinks
            float m = -INFINITY, l = 0.f, base = 0.f, limit = -INFINITY;
            // a query with an infinity or a NaN answers NaN: its negative scores would look like masked ones. A thread looks its own over
            uint32_t most = 0;
            pr_wait(smem_at(&q_full[half]), (uint32_t) (n_q & 1), p.polls, dead);
            __syncwarp();
#pragma unroll
            for (int x = 0; x < HD / 8; x++) {
                uint4 f;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(f.x), "=r"(f.y), "=r"(f.z), "=r"(f.w) : "r"(q_s + half * QB + (x >> 3) * SUB + row * 128 + (((x & 7) ^ (row & 7)) << 4)) : "memory");
                most = __vmaxu2(most, __vmaxu2(__vmaxu2(f.x & 0x7fff7fffu, f.y & 0x7fff7fffu), __vmaxu2(f.z & 0x7fff7fffu, f.w & 0x7fff7fffu)));
            }
            const bool bad = in && wild<T>(most);
            const bool any_bad = __any_sync(0xffffffffu, bad);
            if (lane == 0) pr_arrive(smem_at(&q_empty[half]));
            n_q++;
            const bool odd = any_bad || turned;
            for (int t = 2 * g.t0; t < 2 * g.t1; t++, n_s++) {
                const int pos = step_at(g.sp, t >> 1) * PR_KV + 64 * (t & 1);
                const uint32_t at = my_s + 64 * (n_s & 1);
                pr_wait(smem_at(&s_full[half][n_s & 1]), (uint32_t) (n_s >> 1 & 1), p.polls, dead);
                __syncwarp();
                pr_fence_after();
                const unsigned there = there_s[(g.n0 + (t >> 1) - g.t0) & 3] >> (4 * (t & 1)) & 15u;
                uint32_t r[64];
                pr_ld64(at, r);
                if (odd || there != 15u || pos + 63 > all_see_hi || (pos < all_see_lo && pos + 63 >= a.sinks)) {
                    if (any_bad) {                                         // every score as good as another: whether it sees anything is told by the sum of weights
#pragma unroll
                        for (int x = 0; x < 64; x++) r[x] = bad ? 0 : r[x];
                    }
                    if (turned) {
#pragma unroll
                        for (int x = 0; x < 64; x++) r[x] ^= 0x80000000u;
                    }
                    // what a column does not see goes to -infinity: a bit a token of what it sees, up to its position, behind the window's beginning or among the first ones, on pages that are there
                    const uint64_t pages = (there & 1 ? 0xffffull : 0) | (there & 2 ? 0xffffull << 16 : 0) | (there & 4 ? 0xffffull << 32 : 0) | (there & 8 ? 0xffffull << 48 : 0);
                    const uint64_t seen = first_bits(top_pos - pos + 1) & (~first_bits(low_pos - pos + 1) | first_bits(a.sinks - pos)) & pages;
#pragma unroll
                    for (int x = 0; x < 64; x++) r[x] = seen >> x & 1 ? r[x] : 0xff800000u;
                }
                float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
                for (int x = 0; x < 64; x += 4) {
                    x0 = fmaxf(x0, fmaxf(__uint_as_float(r[x]), __uint_as_float(r[x + 1])));
                    x1 = fmaxf(x1, fmaxf(__uint_as_float(r[x + 2]), __uint_as_float(r[x + 3])));
                }
                const float high = in ? fmaxf(x0, x1) : -INFINITY, score = high == -INFINITY ? high : high * factor;      // (a box's columns behind the sequence's rows, which others write, move no base)
                if (__any_sync(0xffffffffu, score > limit)) {
                    const float top = fmaxf(m, score - p16_lift<T>), down = top > m ? exp2_fast(m - top) : 1.f;
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
                    limit = top + (p16_lift<T> + P_PASS);
                    l *= down;
                }
                const uint64_t by = two(factor, factor), less = two(-base, -base);
                uint64_t sum = 0;
                uint32_t w[32];
#pragma unroll
                for (int x = 0; x < 64; x += 2) {
                    const float2 y = split(fma2(two(__uint_as_float(r[x]), __uint_as_float(r[x + 1])), by, less));
                    const float2 z = (x >> 1 & 7) < P16_EIGHTHS ? exp2_pair(y) : make_float2(exp2_fast(y.x), exp2_fast(y.y));
                    sum = add2(sum, two(z.x, z.y));
                    w[x / 2] = pair_of<T>(z.x, z.y);
                }
                pr_st32(at, w);
                l += split(sum).x + split(sum).y;
                pr_st_wait();
                pr_fence_before();
                __syncwarp();
                if (lane == 0) pr_arrive(smem_at(&p_full[half][n_s & 1]));
            }
            if (bad && l != 0.f) l = NAN;
            // the next segment's queries before this one's results: its first scores are made while these are written
            Segment16 then;
            more = next(then);
            if (more && !by_box) queries(then);
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
    } else {
        regs_less<72>();
        if (warp == 8) {
            // a lane brings its tokens of a tile: a page's, or 128 of a longer page's
            const int log2 = min(c.page_log2, 7), pieces = PR_KV >> log2;
            int n = 0;                                                     // tiles so far
            for (Segment16 g; segment(g);) {
                const auto page_of = [&](int t) { return lane < pieces && t < g.t1 ? page_at(c, g.q.slot, min(step_at(g.sp, t) * PR_KV + (lane << log2), c.max_pages << c.page_log2)) : -1; };
                int page = page_of(g.t0);
                for (int t = g.t0; t < g.t1; t++, n++) {
                    const int stage = n & 1, then = page_of(t + 1);
                    const uint32_t round = (uint32_t) (n >> 1), found = __ballot_sync(0xffffffffu, page >= 0), there = __ballot_sync(0xffffffffu, lane < 8 && (found >> (lane >> (log2 - 4)) & 1));
                    const int token = (step_at(g.sp, t) * PR_KV + (lane << log2)) & ((1 << c.page_log2) - 1), z = page >= 0 ? page : c.n_pages;
#pragma unroll
                    for (int side = 0; side < 2; side++) {
                        const uint32_t full = smem_at(side ? &v_full[stage] : &k_full[stage]), dst = (side ? v_s : k_s) + stage * KVB + (uint32_t) (lane << log2) * 128;
                        if (n >= 2) pr_wait(smem_at(side ? &v_empty[stage] : &k_empty[stage]), (round - 1) & 1, p.polls, dead);
                        dead = __any_sync(0xffffffffu, dead);
                        if (!dead) {
                            if (lane == 0) {
                                if (side == 0) there_s[n & 3] = there;
                                mbar_expect(full, KVB);
                            }
                            __syncwarp();
                            if (lane < pieces)
#pragma unroll
                                for (int d = 0; d < HD / 64; d++) tma_side(dst + d * SUB, &map, full, 64 * d, token, g.head, side, z);
                        }
                    }
                    page = then;
                }
            }
            for (int i = max(0, n - 2); i < n; i++) {                      // the last tiles are let go: their commits arrive while the block's shared memory is its own
                pr_wait(smem_at(&k_empty[i & 1]), (uint32_t) (i >> 1 & 1), p.polls, dead);
                pr_wait(smem_at(&v_empty[i & 1]), (uint32_t) (i >> 1 & 1), p.polls, dead);
            }
        } else if (warp == 11) {
            // queries of the next segment as soon as the last scores of the one before are made
            int n_q[2] = {0, 0};
            for (Segment16 g; by_box && segment(g);)
                for (int half = 0; half < g.halves; half++) {
                    const int use = half ? n_q[1]++ : n_q[0]++;
                    if (use) pr_wait(smem_at(&q_empty[half]), (uint32_t) ((use - 1) & 1), p.polls, dead);
                    __syncwarp();
                    if (pr_elect() && !dead) {
                        mbar_expect(smem_at(&q_full[half]), QB);
#pragma unroll
                        for (int d = 0; d < HD / 64; d++)
                            tma_queries(q_s + half * QB + d * SUB, &q_map, smem_at(&q_full[half]), 64 * d, g.head * a.group, g.q.begin + (g.ct * PR_COLS + half * 128) / a.group);
                    }
                }
            for (int half = 0; half < 2; half++)                           // as with the last tiles
                if (n_q[half]) pr_wait(smem_at(&q_empty[half]), (uint32_t) ((n_q[half] - 1) & 1), p.polls, dead);
        } else {
            const int half = warp - 9;
            int n = 0, n_q = 0, n_p = 0;                                   // tiles, segments and steps of this half so far
            for (Segment16 g; segment(g);) {
                const int tiles = g.t1 - g.t0, steps = 2 * tiles;
                if (pr_elect()) {
                    if (half < g.halves) {
                        const auto scores = [&](int step) {                // S = Q K^T of 64 tokens
                            const int turn = step & 1;
#pragma unroll
                            for (int k = 0; k < HD / 16; k++)
                                pr_mma_ss(t_s + half * 128 + 64 * turn, PR_DESC | (uint64_t) ((q_s + half * QB + (k >> 2) * SUB) >> 4) + 2 * (k & 3),
                                          PR_DESC | (uint64_t) ((k_s + (n + (step >> 1) & 1) * KVB + (k >> 2) * SUB + turn * (SUB / 2)) >> 4) + 2 * (k & 3), p16_idesc<T>(64, false), k > 0);
                            pr_commit(smem_at(&s_full[half][turn]));
                            if (step == steps - 1) pr_commit(smem_at(&q_empty[half]));
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
                            if (turn == 0) {                               // (a wait for what is there takes 130 clocks: while P is being made)
                                pr_wait(smem_at(&v_full[stage]), (uint32_t) (now >> 1 & 1), p.polls, dead);
                                if (step + 2 < steps) pr_wait(smem_at(&k_full[after]), (uint32_t) ((now + 1) >> 1 & 1), p.polls, dead);
                            }
                            pr_wait(smem_at(&p_full[half][turn]), (uint32_t) ((n_p + step) >> 1 & 1), p.polls, dead);
                            pr_fence_after();
                            if (!dead) {
#pragma unroll
                                for (int k = 0; k < 4; k++)
                                    pr_mma_ts(t_o + half * HD, t_s + half * 128 + 64 * turn + 8 * k, P16_V_DESC | (uint64_t) ((v_s + stage * KVB + turn * (SUB / 2) + k * 2048) >> 4), p16_idesc<T>(HD, true),
                                              step > 0 || k > 0);
                                pr_commit(smem_at(&o_full[half][turn]));
                                if (turn == 1) pr_commit(smem_at(&v_empty[stage]));
                            }
                            if (step + 2 < steps) {
                                if (!dead) {
                                    scores(step + 2);
                                    if (turn == 1) pr_commit(smem_at(&k_empty[after]));
                                }
                            }
                        }
                    } else {                                               // no columns here: the tiles are let go as they come
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
    }
    if (dead) atomicExch_system(p.err, 1);
    pr_fence_before();
    if (__syncthreads_or(dead))                                            // nobody issues any more: products and copies under way end before shared and tensor memory are given back
        for (int j = 0; j < 1000; j++) __nanosleep(1000);
    if (warp == 8) {
        pr_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem));
    }
}

// a block 32 columns of a unit that blocks shared: adds its parts, four on their way at a time and four blocks an SM (eight and two: 1000 rows behind 5000
// positions, whose parts are 38 MB, 15 us for 10). A lane is a column, a warp has every eighth group of 4 dims
template <int HD, typename T>
__global__ void __launch_bounds__(256, 4) k_kv16_prompt_join(const PromptArgs p) {
    constexpr int X = HD / 32, PAD = HD + 4, BATCH = 4;
    __shared__ __align__(16) float sums[32 * PAD];
    const AttendArgs & a = p.a;
    const Cache & c = a.c;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x / (PR_COLS / 32), c0 = blockIdx.x % (PR_COLS / 32) * 32, head = blockIdx.y;
    // the plan is done with: the kernel in front waited for it before it let this one begin. Its own results are behind the wait, for which blocks without work stay too
    Entry n = {};
    int cols = 0, w0 = 0, w1 = 0;
    if (e < p.first[1]) {
        n = p.entries[e];
        const int len = n.n + P16_OVER, per = p.first[0];
        cols = min(PR_COLS, n.count * a.group - n.ct * PR_COLS);
        const long long u0 = a.before[e] + (long long) head * len;
        w0 = (int) quotient(u0 + P16_OVER, per);
        w1 = (int) quotient(u0 + len - 1, per);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (c0 >= cols || w0 == w1) return;
    const bool in = c0 + lane < cols;                              // (others were not stored)
    float m = -INFINITY, l = 0.f, o[X][4] = {};
    for (int w = w0; w <= w1; w += BATCH) {
        float2 ml[BATCH];
        float4 v[BATCH][X];
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            const size_t part = 2 * (size_t) (w + i) + (w + i == w0 ? 1 : 0);
            const bool there = in && w + i <= w1;
            ml[i] = there ? *reinterpret_cast<const float2 *>(a.ml + (part * PR_COLS + c0 + lane) * 2) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int x = 0; x < X; x++)
                v[i][x] = there ? reinterpret_cast<const float4 *>(a.part + part * PR_COLS * HD)[(size_t) (warp + 8 * x) * PR_COLS + c0 + lane] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < BATCH; i++) top = fmaxf(top, ml[i].x);
        const float base = top == -INFINITY ? 0.f : top, old = exp2_fast(m - base);
        l *= old;
#pragma unroll
        for (int x = 0; x < X; x++) { o[x][0] *= old; o[x][1] *= old; o[x][2] *= old; o[x][3] *= old; }
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            const float by = exp2_fast(ml[i].x - base);
            l = fmaf(ml[i].y, by, l);
#pragma unroll
            for (int x = 0; x < X; x++) {
                o[x][0] = fmaf(v[i][x].x, by, o[x][0]); o[x][1] = fmaf(v[i][x].y, by, o[x][1]);
                o[x][2] = fmaf(v[i][x].z, by, o[x][2]); o[x][3] = fmaf(v[i][x].w, by, o[x][3]);
            }
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

}  // namespace srv
}  // namespace b200
