// serve_kv16.cuh — the paged cache of 16-bit keys and values, and attention of few rows of many sequences over it (sm_100a).
//
// A page is [2][n_head_kv][page_tokens][head_dim] numbers of the pool's type (bfloat16 or fp16): keys, then values. A token with an infinity or a NaN in a head's key or value (one that the
// type cannot hold among them) stands as a key of NaN and a value of 0: who sees the token answers NaN for the head, nobody else does, and values in the cache are always finite (a masked
// position's weight 0 may be multiplied with them).
// A row at position p sees the positions j <= p that have a page; under a window those with j > p - window or j < sinks.
//
// Few rows: as over the 4-bit cache (serve_attn.cuh), a unit of work is 8 NT columns (a column is a row and a query head of one KV head) over steps of 32 tokens. All units' steps stand in one
// line that is cut evenly over the warps of the grid; a warp walks its piece alone, the running maximum and sum of the soft-max in registers, and leaves partial results of a unit that others
// share for k_kv4_join. Under a window a unit's steps are those of the first tokens and those of the window, side by side.
//   S^T = K Q^T: 16 tokens of K by ldmatrix are the A operand of mma.sync, the columns the B operand; O^T += V^T P^T with V by ldmatrix.trans, P^T from S^T by movmatrix.
// A step (K and V of 32 tokens, 128 head_dim bytes) comes by one TMA box for each 16 tokens and 64 dims, with the 128-byte swizzle that ldmatrix reads without bank conflicts; a page that is
// absent is a box outside the pool, which reads 0. Every warp has a ring of its own, two steps ahead.
// P = hi + lo in two numbers of the type: 16 and 22 bits of a weight, so that results are as good as their own rounding (one number of 8 bits would be another rounding of the result's size;
// the second product hides behind the loads). Sums are fp32; of fp16 P_LIFT and P_PASS as in serve_attn.cuh, of bfloat16 see p16_lift.
// Measured with 32 query heads on 8 of 128, calls one after another on inputs that change: HBM bounds long contexts (48 sequences of 90 to 4090 tokens, 410 MB, 74 us, 86 % of the copy rate over the whole call;
// one of 20 000, 82 MB, 23 us); one launch of clusters 5.8 us at one sequence of 333 tokens, 9.1 at 61 under a window of 1000 with 4 sinks (8 heads on 2 of 64), of which 5 are the launch and the way
// slot -> length -> page -> box -> products -> the cluster's meetings.
#pragma once
#include "serve_attn.cuh"
#include "serve_tma.cuh"
#include <cooperative_groups.h>
#include <type_traits>

namespace b200 {
namespace srv {

// The first kernel of a call stands ready behind the work in front of it (programmatic launch), waits for that before it touches any memory of the call, and only then lets the kernel behind it
// begin, which may read ahead of its own wait what the call was given. Rows of 4 sequences written and attended to, calls one after another: 12.3 us without, 7.7 so.
constexpr int A16_WARPS = 4, A16_STAGES = 3, A16_STEP = 32, A16_CLUSTER = 8;      // A16_STAGES: a warp
__host__ __device__ constexpr int a16_stage_bytes(int hd) { return A16_STEP * 4 * hd; }
__host__ __device__ constexpr size_t a16_ring_bytes(int hd) { return (size_t) A16_WARPS * A16_STAGES * a16_stage_bytes(hd); }

// what the base of a weight 2^(score - base) is below the largest score (serve_attn.cuh). bfloat16 keeps its 8 bits at any size, so it needs no lift; but its values go up to fp32's largest, and so
// would sums of values with weights above 1. With weights of 2^-38 at the largest score, 2^-30 until the base moves, those of the 2^30 tokens that a slot can have sum up to less than 1, and no sum of
// values passes the largest value. At the other end, what of a result is below 2^-88 may be lost.
template <typename T> constexpr float p16_lift = std::is_same<T, __half>::value ? P_LIFT : -30.f - P_PASS;

// steps of 2^log2 tokens that the rows a .. b of a sequence see: `head` of them from position 0, the others from step lo on
struct Steps { int head, lo, n; };
__device__ __forceinline__ Steps steps_of(const Cache & c, const Seq & q, int window, int sinks, int a, int b, int log2) {
    const int last = min(q.held + b, (c.max_pages << c.page_log2) - 1), first = window > 0 ? max(0, q.held + a - window + 1) : 0;
    if (q.slot < 0) return Steps{0, 0, 1};
    Steps s;
    s.lo = first >> log2;
    s.head = window > 0 ? min((int) (((long long) min(sinks, last + 1) + (1 << log2) - 1) >> log2), s.lo) : 0;
    s.n = max(1, s.head + (last < first ? 0 : (last >> log2) - s.lo + 1));
    return s;
}
__device__ __forceinline__ int step_at(const Steps & s, int i) { return i < s.head ? i : i - s.head + s.lo; }

template <typename T> __device__ __forceinline__ void mma_of(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value) mma_16816(d, a, b0, b1);
    else asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS> __device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    if constexpr (TRANS) asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
    else asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T> __device__ __forceinline__ uint32_t pair_of(float x, float y) {
    if constexpr (std::is_same<T, __half>::value) return as_u(__floats2half2_rn(x, y));
    else { const __nv_bfloat162 p = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t *>(&p); }
}
template <typename T> __device__ __forceinline__ float2 floats_of(uint32_t p) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(as_h2(p));
    else return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}
// whether one of a pair is an infinity or a NaN
template <typename T> __device__ __forceinline__ bool wild(uint32_t p) {
    constexpr uint32_t M = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    return (p & M) == M || (p >> 16 & M) == M;
}

// what a warp holds of a unit: its columns' sums of values, largest scores less the lift and sums of weights. A lane has columns 2 tq, 2 tq + 1 of each eight and the dims 16 k + g, + 8
template <int HD, int NT> struct Piece16 { float o[NT][HD / 16][4], m[NT][2], l[NT][2]; };
// CW warps go over the same steps with columns of their own: one of them asks for the steps, all tell when they are done with one. Of a ring: where its stages, the barriers that tell a stage full
// (and, where it is shared, empty) stand, and steps that were asked for and used so far: stage n % (A16_STAGES CW), phase n / (A16_STAGES CW)
struct Ring16 { uint32_t at, full, empty; int n_fill, n_use; };

// steps t0 .. t1 - 1 of the columns ct (a warp's own) of a sequence and KV head
template <int HD, int NT, int CW, typename T>
__device__ __forceinline__ void attend_piece(const AttendArgs & a, const CUtensorMap & map, const Seq & q, const Steps & sp, int ct, int head, int t0, int t1, Ring16 & ring, bool asks, uint32_t polls, bool & dead,
                                             Piece16<HD, NT> & out) {
    constexpr int STAGES = A16_STAGES * CW, AHEAD = CW == 1 ? STAGES - 1 : STAGES - 2;         // (of a shared ring a step less, so that the one that asks waits for nobody)
    constexpr int COLS = 8 * NT, KS = HD / 16, STAGE = a16_stage_bytes(HD), HALF = 8192;        // HALF: 64 dims of a step; of it 4096 for 16 tokens, keys and values of 2048 each
    const int lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    const Cache & c = a.c;
    float (&o)[NT][KS][4] = out.o;
    float (&m)[NT][2] = out.m;
    float (&l)[NT][2] = out.l;
    // the columns' queries, B operand of K Q^T: lane (g, tq) holds column g's dims 16 k + 2 tq, + 1 and those 8 further on
    uint32_t qf[NT][KS][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int col = ct * COLS + 8 * n + g, i = col / a.group, h = head * a.group + col - i * a.group;
        const T * qp = static_cast<const T *>(a.q) + (q.begin + i) * a.q_row + h * a.q_head + 2 * tq;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                qf[n][k][j] = 0;
                if (i >= q.count) continue;
                if (a.q_whole) qf[n][k][j] = *reinterpret_cast<const uint32_t *>(qp + 16 * k + 8 * j);
                else { const uint16_t * u = reinterpret_cast<const uint16_t *>(qp + 16 * k + 8 * j); qf[n][k][j] = u[0] | (uint32_t) u[1] << 16; }
            }
    }
    // steps on their way: AHEAD of the one in hand. Lanes hold the next 32 pages of the slot
    const bool idle = (int64_t) ct * COLS >= (int64_t) q.count * a.group;      // (of a shared ring: a warp without columns)
    int next = t0, pages_from = -64, my_page = -1;
    uint32_t there = 0;                                        // two bits a step that was asked for: which of its halves have a page. The newest lowest
    const auto fetch = [&]() {
        there <<= 2;
        if (next < t1) {
            const int pos = step_at(sp, next) << 5, pi = pos >> c.page_log2, pi_b = (pos + 16) >> c.page_log2;
            if (pi < pages_from || pi_b - pages_from > 31) { pages_from = pi; my_page = page_at(c, q.slot, min(pi + lane, c.max_pages) << c.page_log2); }
            const int page_a = __shfl_sync(0xffffffffu, my_page, pi - pages_from), page_b = __shfl_sync(0xffffffffu, my_page, pi_b - pages_from);
            there |= (uint32_t) (page_a >= 0) | (uint32_t) (page_b >= 0) << 1;
            const int stage = ring.n_fill % STAGES;
            if (CW > 1 && asks && ring.n_fill >= STAGES) mbar_wait(ring.empty + 8 * stage, (uint32_t) ((ring.n_fill / STAGES - 1) & 1), polls, dead);
            if (asks && lane == 0 && !dead) {
                const int mask = (1 << c.page_log2) - 1;
                const uint32_t bar = ring.full + 8 * stage, dst = ring.at + (uint32_t) (stage * STAGE);
                mbar_expect(bar, STAGE);
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int h = 0; h < HD / 64; h++)
                        tma_box(dst + h * HALF + u * 4096, &map, bar, 64 * h, (pos + 16 * u) & mask, head, u ? (page_b >= 0 ? page_b : c.n_pages) : (page_a >= 0 ? page_a : c.n_pages));
            }
            ring.n_fill++;
            next++;
        }
    };
    __syncwarp();                                              // nobody still reads the ring for the piece before
#pragma unroll
    for (int i = 0; i < AHEAD; i++) fetch();
    int p_hi[NT][2];                                           // last position that the lane's two columns of S^T see; -1: no column
#pragma unroll
    for (int n = 0; n < NT; n++) {
        // a query with an infinity has no soft-max that is a number: all NaN, since negative scores would look like masked ones
        bool bad = false;
#pragma unroll
        for (int k = 0; k < KS; k++) bad = bad || wild<T>(qf[n][k][0]) || wild<T>(qf[n][k][1]);
        const unsigned any = __ballot_sync(0xffffffffu, bad) >> (4 * g) & 15u;
#pragma unroll
        for (int k = 0; k < KS; k++) if (any) qf[n][k][0] = qf[n][k][1] = 0x7fff7fffu;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int cc = ct * COLS + 8 * n + 2 * tq + j;
            p_hi[n][j] = cc / a.group < q.count ? q.held + cc / a.group : -1;
        }
    }
    const int row_lo = ct * COLS / a.group, row_hi = min(q.count - 1, (ct * COLS + COLS - 1) / a.group);
    const int all_see_hi = q.held + row_lo, all_see_lo = a.window > 0 ? q.held + row_hi - a.window + 1 : 0;   // positions that every column sees
    float base[NT][2], limit[NT][2];       // base: what is taken off scores, m or 0; limit: where they move
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int j = 0; j < 2; j++) { m[n][j] = limit[n][j] = -INFINITY; l[n][j] = base[n][j] = 0.f; }
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[n][k][j] = 0.f;
    }
    const uint32_t k_lane = (uint32_t) ((lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4));
    const uint32_t v_lane = (uint32_t) (2048 + ((lane & 7) + ((lane >> 4) << 3)) * 128 + (((lane >> 3 & 1) ^ (lane & 7)) << 4));
#pragma unroll 1
    for (int t = t0; t < t1; t++) {
        const int stage = ring.n_use % STAGES;
        mbar_wait(ring.full + 8 * stage, (uint32_t) (ring.n_use / STAGES & 1), polls, dead);
        ring.n_use++;
        dead = __any_sync(0xffffffffu, dead);                  // (and all lanes are done with the step before)
        if (dead) return;
        fetch();
        const uint32_t step = ring.at + (uint32_t) (stage * STAGE);
        const uint32_t both = there >> 2 * AHEAD & 3;
        const auto leave = [&]() {
            if (CW > 1) {
                __syncwarp();
                if (lane == 0) mbar_arrive(ring.empty + 8 * stage);
            }
        };
        if (both == 0 || (CW > 1 && idle)) { leave(); continue; }
        const int pos = step_at(sp, t) << 5;
        float st[2][NT][4];
#pragma unroll
        for (int u = 0; u < 2; u++) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) st[u][n][j] = 0.f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                uint32_t f[4];
                ldsm4<false>(f, step + (k >> 2) * HALF + u * 4096 + (k_lane ^ (uint32_t) ((k & 3) << 5)));
#pragma unroll
                for (int n = 0; n < NT; n++) mma_of<T>(st[u][n], f, qf[n][k][0], qf[n][k][1]);
            }
        }
        bool more = false;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) { st[0][n][j] *= a.scale_log2; st[1][n][j] *= a.scale_log2; }
        // rows of S^T: tokens g and g + 8 of each 16
        if (pos + 31 > all_see_hi || (pos < all_see_lo && pos + 31 >= a.sinks) || both != 3) {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int p = pos + g + 16 * u + 8 * (j >> 1), top = p_hi[n][j & 1];
                        if (p > top || (a.window > 0 && p <= top - a.window && p >= a.sinks) || !(both >> u & 1)) st[u][n][j] = -INFINITY;
                    }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 2; j++) more = more || fmaxf(fmaxf(st[0][n][j], st[0][n][j + 2]), fmaxf(st[1][n][j], st[1][n][j + 2])) > limit[n][j];
        // base moves when a score passes the largest so far by 2^P_PASS
        if (__any_sync(0xffffffffu, more)) {
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float x = fmaxf(fmaxf(st[0][n][j], st[0][n][j + 2]), fmaxf(st[1][n][j], st[1][n][j + 2]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    const float top = fmaxf(m[n][j], x - p16_lift<T>), down = top > m[n][j] ? exp2_fast(m[n][j] - top) : 1.f;
                    m[n][j] = top;
                    base[n][j] = top == -INFINITY ? 0.f : top;
                    limit[n][j] = top + (p16_lift<T> + P_PASS);
                    l[n][j] *= down;
#pragma unroll
                    for (int k = 0; k < KS; k++) { o[n][k][j] *= down; o[n][k][j + 2] *= down; }
                }
        }
        uint32_t hi[2][NT][2], lo[2][NT][2];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    st[u][n][j] = exp2_fast(st[u][n][j] - base[n][j & 1]);
                    l[n][j & 1] += st[u][n][j];
                }
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint32_t p = pair_of<T>(st[u][n][2 * j], st[u][n][2 * j + 1]);
                    const float2 f = floats_of<T>(p);
                    hi[u][n][j] = transposed(p);
                    lo[u][n][j] = transposed(pair_of<T>(st[u][n][2 * j] - f.x, st[u][n][2 * j + 1] - f.y));
                }
            }
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int k = 0; k < KS; k++) {
                uint32_t f[4];
                ldsm4<true>(f, step + (k >> 2) * HALF + u * 4096 + (v_lane ^ (uint32_t) ((k & 3) << 5)));
#pragma unroll
                for (int n = 0; n < NT; n++) { mma_of<T>(o[n][k], f, hi[u][n][0], hi[u][n][1]); mma_of<T>(o[n][k], f, lo[u][n][0], lo[u][n][1]); }
            }
        leave();
    }
    // sums over the tokens, which lie over the lanes' g
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 4);
            l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 8);
            l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 16);
        }
}

// boxes: arrivals that tell a step there, 1, or more than come (b200_kv4_drill)
template <int HD, int NT, typename T>
__global__ void __launch_bounds__(A16_WARPS * 32, 1) k_kv16_attend(const AttendArgs a, const __grid_constant__ CUtensorMap map, int * err, uint32_t polls, int boxes) {
    constexpr int COLS = 8 * NT, KS = HD / 16, STAGE = a16_stage_bytes(HD);
    extern __shared__ uint8_t a16_raw[];
    __shared__ long long sums[A16_WARPS];
    __shared__ __align__(8) uint64_t full_s[A16_WARPS][A16_STAGES];
    const uint32_t smem = (smem_at(a16_raw) + 1023u) & ~1023u;
    long long * before = reinterpret_cast<long long *>(a16_raw + (smem - smem_at(a16_raw)) + a16_ring_bytes(HD));       // [n_seq + 1]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3;
    const Cache & c = a.c;
    if (lane == 0) {
        for (int i = 0; i < A16_STAGES; i++) mbar_init(smem_at(&full_s[warp][i]), boxes);
        mbar_init_done();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // steps in front of each sequence
    {
        constexpr int THREADS = A16_WARPS * 32, BATCH = 4;
        for (int b0 = tid; b0 < c.n_seq; b0 += THREADS * BATCH) {              // (slot, held, first: dependent reads, of four sequences at a time)
            Seq q[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) q[i] = seq_at(c, min(b0 + i * THREADS, c.n_seq - 1));
#pragma unroll
            for (int i = 0; i < BATCH; i++)
                if (b0 + i * THREADS < c.n_seq)
                    before[b0 + i * THREADS] = q[i].count ? (long long) col_tiles(q[i], a.group, COLS) * c.n_kv * (steps_of(c, q[i], a.window, a.sinks, 0, q[i].count - 1, 5).n + AT_OVER) : 0;
        }
        __syncthreads();
        const int each = (c.n_seq + THREADS - 1) / THREADS, s0 = min(c.n_seq, tid * each), s1 = min(c.n_seq, s0 + each);
        long long mine = 0;
        for (int s = s0; s < s1; s++) { const long long n = before[s]; before[s] = mine; mine += n; }
        long long up = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, up, d); if (lane >= d) up += x; }
        if (lane == 31) sums[warp] = up;
        __syncthreads();
        long long off = up - mine;
        for (int w = 0; w < warp; w++) off += sums[w];
        for (int s = s0; s < s1; s++) before[s] += off;
        if (tid == THREADS - 1) before[c.n_seq] = off + mine;
        __syncthreads();
    }
    const long long total = before[c.n_seq];
    const int n_warps = (int) gridDim.x * A16_WARPS;
    const long long per = max(1ll, quotient(total + n_warps - 1, n_warps));
    if (blockIdx.x == 0) {
        for (int s = tid; s <= c.n_seq; s += A16_WARPS * 32) a.before[s] = before[s];
        if (tid == 0) a.before[c.n_seq + 1] = per;
    }
    const int me = warp * (int) gridDim.x + (int) blockIdx.x;      // neighbouring pieces on different SMs
    Ring16 ring = {smem + (uint32_t) (warp * A16_STAGES * STAGE), smem_at(&full_s[warp][0]), 0, 0, 0};
    bool dead = false;
    long long at = me * per;
    const long long end = min(total, at + per);
    while (at < end) {
        int s = 0;
        for (int hi = c.n_seq; hi - s > 1;) { const int mid = (s + hi) >> 1; if (before[mid] <= at) s = mid; else hi = mid; }
        const Seq q = seq_at(c, s);
        const Steps sp = steps_of(c, q, a.window, a.sinks, 0, q.count - 1, 5);
        const long long x = at - before[s];
        const int len = sp.n + AT_OVER, unit = (int) quotient(x, len), from = (int) (x - (long long) unit * len), to = (int) min((long long) len, from + (end - at));
        const int ct = unit / c.n_kv, head = unit - ct * c.n_kv, t0 = max(0, from - AT_OVER), t1 = to - AT_OVER;
        at += to - from;
        if (t1 <= 0) continue;
        Piece16<HD, NT> w;
        attend_piece<HD, NT, 1, T>(a, map, q, sp, ct, head, t0, t1, ring, true, polls, dead, w);
        if (dead) break;
        const bool whole = t0 == 0 && t1 == sp.n;
        const size_t slot = 2 * (size_t) me + (t0 == 0 ? 1 : 0);
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int in_tile = 8 * n + 2 * tq + j, col = ct * COLS + in_tile, i = col / a.group, h = head * a.group + col - i * a.group;
                if (i >= q.count) continue;
                if (whole) {
                    const float inv = w.l[n][j] != 0.f ? 1.f / w.l[n][j] : 0.f;
                    T * y = static_cast<T *>(a.out) + ((size_t) (q.begin + i) * c.n_kv * a.group + h) * HD + g;
#pragma unroll
                    for (int k = 0; k < KS; k++) { y[16 * k] = from_f<T>(w.o[n][k][j] * inv); y[16 * k + 8] = from_f<T>(w.o[n][k][j + 2] * inv); }
                } else {
                    float * y = a.part + (slot * COLS + in_tile) * HD + g;
#pragma unroll
                    for (int k = 0; k < KS; k++) { y[16 * k] = w.o[n][k][j]; y[16 * k + 8] = w.o[n][k][j + 2]; }
                    if (g == 0) *reinterpret_cast<float2 *>(a.ml + (slot * COLS + in_tile) * 2) = make_float2(w.m[n][j], w.l[n][j]);
                }
            }
    }
    if (dead) {                                                    // the call's results are worthless; its own copies end before the block gives its memory back
        if (lane == 0) atomicExch_system(err, 1);
        for (int j = 0; j < 1000; j++) __nanosleep(1000);
    }
}

// Few sequences of bounded length, up to 64 columns: with more than 16 two or four warps (CW) go over the same steps with 16 columns each, so that keys and values are read once. (In the line of pieces
// such groups are slower than tcgen05: a step is one chain of 2200 clocks, and a block has one or two of them under way. 48 ragged sequences of 20 columns 121 us and 96, 6 long ones of 40 270 and 100.) A cluster of blocks a unit, its warps share the unit's steps evenly and the blocks add what they have through one another's shared memory. One launch, no workspace
template <int HD, int NT, int CW, typename T>
__global__ void __launch_bounds__(A16_WARPS * 32, 1) k_kv16_attend_unit(const AttendArgs a, const __grid_constant__ CUtensorMap map, int * err, uint32_t polls, int boxes) {
    constexpr int COLS = 8 * NT, ALL = COLS * CW, KS = HD / 16, STAGE = a16_stage_bytes(HD), PAD = HD + 4, GROUPS = A16_WARPS / CW, STAGES = A16_STAGES * CW;
    extern __shared__ uint8_t a16_raw[];
    __shared__ __align__(8) uint64_t full_s[GROUPS][STAGES], empty_s[GROUPS][STAGES];
    __shared__ __align__(8) float ml_s[GROUPS][ALL][2], ml_b[ALL][2];
    namespace cg = cooperative_groups;
    cg::cluster_group cl = cg::this_cluster();
    const uint32_t smem = (smem_at(a16_raw) + 1023u) & ~1023u;
    float * parts = reinterpret_cast<float *>(a16_raw + (smem - smem_at(a16_raw)));        // [groups][ALL][PAD], then of the block [ALL][PAD], over the ring when it is done with
    static_assert((GROUPS + 1) * ALL * PAD * 4 <= a16_ring_bytes(HD), "parts stand in the ring");
    float * sums = parts + GROUPS * ALL * PAD;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, cw = warp % CW, group = warp / CW, g = lane >> 2, tq = lane & 3, rank = (int) cl.block_rank(), blocks = (int) cl.num_blocks();
    const Cache & c = a.c;
    if (lane == 0 && cw == 0) {
        for (int i = 0; i < STAGES; i++) { mbar_init(smem_at(&full_s[group][i]), boxes); mbar_init(smem_at(&empty_s[group][i]), CW); }
        mbar_init_done();
    }
    if (CW > 1) __syncthreads(); else __syncwarp();
    Ring16 ring = {smem + (uint32_t) (group * STAGES * STAGE), smem_at(&full_s[group][0]), smem_at(&empty_s[group][0]), 0, 0};
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int unit = (int) blockIdx.x / blocks, head = unit % c.n_kv, s = unit / c.n_kv;
    const Seq q = seq_at(c, s);
    const Steps sp = steps_of(c, q, a.window, a.sinks, 0, q.count - 1, 5);
    const int all_groups = blocks * GROUPS, me = rank * GROUPS + group, per = sp.n / all_groups, more = sp.n % all_groups, t0 = me * per + min(me, more), t1 = t0 + per + (me < more);
    bool dead = false;
    for (int ct = 0; ct < col_tiles(q, a.group, ALL); ct++) {       // (more than one where a sequence has more rows than max_rows says. The same for all blocks of the cluster)
        Piece16<HD, NT> w;
        attend_piece<HD, NT, CW, T>(a, map, q, sp, ct * CW + cw, head, t0, dead ? t0 : t1, ring, cw == 0, polls, dead, w);
        __syncthreads();                                           // nobody reads the ring any more
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int col = cw * COLS + 8 * n + 2 * tq + j;
                float * y = parts + (group * ALL + col) * PAD + g;
#pragma unroll
                for (int k = 0; k < KS; k++) { y[16 * k] = w.o[n][k][j]; y[16 * k + 8] = w.o[n][k][j + 2]; }
                if (g == 0) { ml_s[group][col][0] = w.m[n][j]; ml_s[group][col][1] = w.l[n][j]; }
            }
        __syncthreads();
        // the block's sum, four dims a thread
        for (int i = tid; i < ALL * HD / 4; i += A16_WARPS * 32) {
            const int col = i / (HD / 4), d = i % (HD / 4) * 4;
            float top = -INFINITY, l = 0.f;
#pragma unroll
            for (int v = 0; v < GROUPS; v++) top = fmaxf(top, ml_s[v][col][0]);
            const float base = top == -INFINITY ? 0.f : top;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int v = 0; v < GROUPS; v++) {
                const float by = exp2_fast(ml_s[v][col][0] - base);
                const float4 y = *reinterpret_cast<const float4 *>(parts + (v * ALL + col) * PAD + d);
                l = fmaf(ml_s[v][col][1], by, l);
                x.x = fmaf(y.x, by, x.x); x.y = fmaf(y.y, by, x.y); x.z = fmaf(y.z, by, x.z); x.w = fmaf(y.w, by, x.w);
            }
            *reinterpret_cast<float4 *>(sums + col * PAD + d) = x;
            if (d == 0) { ml_b[col][0] = top; ml_b[col][1] = l; }
        }
        cl.sync();
        // the blocks', a share of the results each
        const int first = ct * ALL;
        for (int i = rank * A16_WARPS * 32 + tid; i < ALL * HD / 4; i += blocks * A16_WARPS * 32) {
            const int col = i / (HD / 4), d = i % (HD / 4) * 4, r = (first + col) / a.group, h = head * a.group + first + col - r * a.group;
            if (r >= q.count) continue;
            float2 ml[A16_CLUSTER];
            float4 y[A16_CLUSTER];
#pragma unroll
            for (int b = 0; b < A16_CLUSTER; b++) {
                const int o = b < blocks ? b : 0;
                ml[b] = *reinterpret_cast<const float2 *>(cl.map_shared_rank(&ml_b[col][0], o));
                y[b] = *reinterpret_cast<const float4 *>(cl.map_shared_rank(sums + col * PAD + d, o));
            }
            float top = -INFINITY, l = 0.f;
#pragma unroll
            for (int b = 0; b < A16_CLUSTER; b++) top = fmaxf(top, b < blocks ? ml[b].x : -INFINITY);
            const float base = top == -INFINITY ? 0.f : top;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int b = 0; b < A16_CLUSTER; b++)
                if (b < blocks) {
                    const float by = exp2_fast(ml[b].x - base);
                    l = fmaf(ml[b].y, by, l);
                    x.x = fmaf(y[b].x, by, x.x); x.y = fmaf(y[b].y, by, x.y); x.z = fmaf(y[b].z, by, x.z); x.w = fmaf(y[b].w, by, x.w);
                }
            const float inv = l != 0.f ? 1.f / l : 0.f;
            Four<T> f;
            f.v[0] = from_f<T>(x.x * inv); f.v[1] = from_f<T>(x.y * inv); f.v[2] = from_f<T>(x.z * inv); f.v[3] = from_f<T>(x.w * inv);
            *reinterpret_cast<Four<T> *>(static_cast<T *>(a.out) + ((size_t) (q.begin + r) * c.n_kv * a.group + h) * HD + d) = f;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        cl.sync();                                                 // nobody reads this block's any more: boxes may come into the ring again, or the block ends
    }
    if (dead) {
        if (lane == 0) atomicExch_system(err, 1);
        for (int j = 0; j < 1000; j++) __nanosleep(1000);
    }
}

// ---- rows into the cache -----------------------------------------------------------------------------------------------------
template <typename S> struct Row16Src { const S * k; int64_t k_row, k_head; const S * v; int64_t v_row, v_head; bool whole8; };
// eight entries as four pairs of T, each rounded once. wild: one is an infinity or a NaN
template <typename S, typename T> __device__ __forceinline__ void eight_as(const S * p, bool whole, uint32_t (&w)[4]) {
    if (whole) {
        if constexpr (sizeof(S) == 4) {
            const float4 x = reinterpret_cast<const float4 *>(p)[0], y = reinterpret_cast<const float4 *>(p)[1];
            w[0] = pair_of<T>(x.x, x.y); w[1] = pair_of<T>(x.z, x.w); w[2] = pair_of<T>(y.x, y.y); w[3] = pair_of<T>(y.z, y.w);
        } else {
            const uint4 x = *reinterpret_cast<const uint4 *>(p);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
            if constexpr (!std::is_same<S, T>::value)
#pragma unroll
                for (int i = 0; i < 4; i++) { const float2 f = floats_of<S>(w[i]); w[i] = pair_of<T>(f.x, f.y); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = pair_of<T>(to_f(p[2 * i]), to_f(p[2 * i + 1]));
    }
}
// A warp a row and two of its heads (four of 64 dims), 16 bytes a lane; latency bounds few rows (row -> sequence -> slot -> page: 48 of 8 heads 2.2 us), the memory many. Several heads one after the other in a
// warp were slower at all sizes but one: 500 rows of 8 heads of 128 3.4 us for 2.9, 3000 6.2 for 6.4, 8192 13.4 for 12.8, 5200 from fp32 14.9 for 13.7 (62 MB, 4.5 TB/s), 8192 of 2 heads of 64 6.9 for 3.8
template <typename S, typename T, int HD>
__global__ void __launch_bounds__(256) k_kv16_append(const Cache c, const Row16Src<S> src, int parts) {
    constexpr int LANES = HD / 8, PER = 32 / LANES;
    const int64_t item = ((int64_t) blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31, li = lane % LANES, row = (int) (item / parts), head = (int) (item % parts) * PER + lane / LANES;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row >= c.n_rows) return;
    uint32_t k[4] = {}, v[4] = {};
    if (head < c.n_kv) {
        eight_as<S, T>(src.k + row * src.k_row + head * src.k_head + 8 * li, src.whole8, k);
        eight_as<S, T>(src.v + row * src.v_row + head * src.v_head + 8 * li, src.whole8, v);
    }
    const int s = seq_of_row_warp(c, row);
    if (s < 0) return;
    const Seq q = seq_at(c, s);
    const int pos = q.held + row - q.begin, page = page_at(c, q.slot, pos);
    if (page < 0) return;
    const unsigned mine = (LANES == 16 ? 0xffffu : 0xffu) << (lane / LANES * LANES);
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; j++) bad = bad || wild<T>(k[j]) || wild<T>(v[j]);
    if (__ballot_sync(0xffffffffu, bad) & mine)
#pragma unroll
        for (int j = 0; j < 4; j++) { k[j] = 0x7fff7fffu; v[j] = 0; }
    if (head < c.n_kv) {
        uint8_t * to = c.pool + (int64_t) page * c.page_stride + (((int64_t) head << c.page_log2) + (pos & ((1 << c.page_log2) - 1))) * (2 * HD) + 16 * li;
        *reinterpret_cast<uint4 *>(to) = make_uint4(k[0], k[1], k[2], k[3]);
        *reinterpret_cast<uint4 *>(to + ((int64_t) c.n_kv << c.page_log2) * (2 * HD)) = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

}  // namespace srv
}  // namespace b200
