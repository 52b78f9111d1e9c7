// serve_sample.cuh — the draw of next tokens from rows of logits (sm_100a).
//
// A row's tokens are ordered by logit, the lower index first among equals. Each filter keeps a prefix of that order: top-k the first k; top-p, of those, the shortest prefix with at least
// the share p of their weight exp(logit - largest); min-p those of weight at least min_p. Of what all three keep, token i is drawn with weight exp((logit - largest) / temperature): the
// first one in order of index at which the sum exceeds u x total. A filter's edge and the draw are decisions on sums, so weights are whole multiples of 2^-40 from 64-bit exponentials and
// sums of them are exact: no order of summation, and no other split of the row, changes a result.
//
// A cluster of blocks takes a row and holds its slice in shared memory: logits cross HBM once. A histogram of floor(16 x logit), against each block's own largest, tells with one meeting
// of the cluster the row's largest and the bin of the k-th token. Only tokens down to that bin are ordered (a few dozen of 128 k), exactly as the definition says, and the first block
// ends the row with them. For top-p alone counts bound the bins between which its sum is crossed; one sweep sums all weights, those in front of these bins and, in 512 finer bins, those
// between; the tokens of one finer bin are ordered. Then a last sweep sums what is kept, 128 tokens at a time, and the warp in whose tokens the draw falls looks for it. Rows whose edge
// lies among more than 2048 candidates (thousands of equal logits, very large k) are bisected over (logit, index) instead.
//
// Measured with 128 256 logits in fp32, one row / 160 rows (82 MB, 13 us at the copy rate): the largest 6 / 36 us, min-p 8 / 45, top-k 40 10 / 53, no filter 10 / 64, top-p alone 26 / 170.
// Five waves of clusters, two blocks an SM: a wave loads 3000 clocks, and each meeting of a cluster costs it 1200 to 2500 more; then the 64-bit pipe (11 operations a weight) bounds the
// sweeps over all weights.
#pragma once
#include "serve_cache.cuh"
#include <cooperative_groups.h>

namespace b200 {
namespace srv {

namespace cg = cooperative_groups;

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32, SA_BINS = 512, SA_FINE = 512, SA_LIST = 2048, SA_SHORT = SA_THREADS, SA_MAX_CLUSTER = 8, SA_MAX_VOCAB = 1 << 18, SA_SWEEPS = SA_MAX_VOCAB / SA_MAX_CLUSTER / SA_THREADS / 4;
constexpr float SA_PER_NAT = 16.f;
constexpr double SA_ONE = 1099511627776.0;                               // 2^40
typedef unsigned long long u64;

struct SampleArgs {
    const void * logits;
    int64_t row_stride;
    int n_rows, n_vocab, slice;          // slice: entries of a row per block of its cluster
    const float * u, * temperature, * top_p, * min_p;
    const int32_t * top_k;
    int32_t * ids;
    float * logprobs;
};

// 2^40 exp(d steps ln 2 / 16), d <= 0, to the nearest whole number, or 0: y = d steps = n + f with |f| <= 1 / 2, so a table's 2^(n mod 16 / 16), whose 16 entries are the 32 banks of
// shared memory, times 2^(n / 16) times the series of exp(f ln 2 / 16), whose first term left out is below 2^-42. What is left out has its upper word cleared, which adds nothing to 2^52
constexpr double SA_LN = 0.69314718055994530942 / 16;
__constant__ double sa_series[5] = {SA_LN, SA_LN * SA_LN / 2, SA_LN * SA_LN * SA_LN / 6, SA_LN * SA_LN * SA_LN * SA_LN / 24, SA_LN * SA_LN * SA_LN * SA_LN * SA_LN / 120};
__device__ __forceinline__ u64 fixed_weight(double d, double steps, bool in, const double * table) {
    constexpr double WHOLE = 6755399441055744.0, WIDE = 4503599627370496.0;      // 1.5 x 2^52 and 2^52: added, the last bits are a whole number
    const double t = fma(d, steps, WHOLE), f = fma(d, steps, WHOLE - t);
    const int n = __double2loint(t);
    double p = fma(sa_series[4], f, sa_series[3]);
    p = fma(p, f, sa_series[2]);
    p = fma(p, f, sa_series[1]);
    p = fma(p, f, sa_series[0]);
    p = fma(p, f, 1.0) * table[n & 15];
    p = __hiloint2double(in ? __double2hiint(p) + ((n & ~15) << 16) + (40 << 20) : 0, __double2loint(p)) + WIDE;
    return (u64) __double_as_longlong(p) - 0x4330000000000000ull;
}

// (logit, index) as one number: larger is earlier in the order
__device__ __forceinline__ u64 order_key(float v, int i) {                // (-0 as 0, NaN as -infinity)
    const uint32_t b = __float_as_uint(v == v ? v + 0.f : -INFINITY);
    return (u64) (b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t) ~i;
}
__device__ __forceinline__ float key_logit(u64 k) {
    const uint32_t b = (uint32_t) (k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_index(u64 k) { return (int) ~(uint32_t) k; }

template <typename F> __device__ __forceinline__ u64 warp_reduce(u64 x, F f) {
#pragma unroll
    for (int d = 16; d; d >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}
// sums below 2^54 each, as whole numbers of 27 bits
__device__ __forceinline__ u64 warp_sum(u64 x) {
    return (u64) __reduce_add_sync(0xffffffffu, (uint32_t) x & 0x7ffffffu) + ((u64) __reduce_add_sync(0xffffffffu, (uint32_t) (x >> 27)) << 27);
}
struct alignas(128) SampleSmem {
    double table[16];
    u64 red[SA_WARPS], each[SA_MAX_CLUSTER], turn[2][SA_MAX_CLUSTER], sums[SA_MAX_CLUSTER][2];
    u64 answer[4];
    u64 parts[SA_SWEEPS][SA_WARPS];
    float top;                           // the block's largest, and its place among the bins
    int place, n_list;
};
// dynamic shared memory: the list, fine sums, fine counts, bins, the slice
constexpr int SA_FIXED = 8 * SA_LIST + 12 * SA_FINE + 4 * SA_BINS;
// a number of every thread of the cluster, joined; all threads get it
template <typename F> __device__ __forceinline__ u64 cluster_join(cg::cluster_group & cl, SampleSmem & sm, u64 x, u64 none, int & turn, F f) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    x = warp_reduce(x, f);
    __syncthreads();
    if (lane == 0) sm.red[warp] = x;
    __syncthreads();
    if (warp == 0) {
        x = warp_reduce(lane < SA_WARPS ? sm.red[lane] : none, f);
        if (lane < cl.num_blocks()) cl.map_shared_rank(&sm, lane)->turn[turn][cl.block_rank()] = x;
    }
    cl.sync();
    u64 all = none;
    for (unsigned r = 0; r < cl.num_blocks(); r++) all = f(all, sm.turn[turn][r]);
    turn ^= 1;
    return all;
}
// sum over the threads in front of this one, and of the block
__device__ __forceinline__ u64 block_before64(u64 mine, u64 & all, u64 * red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 up = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const u64 x = __shfl_up_sync(0xffffffffu, up, d); if (lane >= d) up += x; }
    __syncthreads();
    if (lane == 31) red[warp] = up;
    __syncthreads();
    u64 part = lane < SA_WARPS ? red[lane] : 0;
#pragma unroll
    for (int d = 1; d < SA_WARPS; d <<= 1) { const u64 x = __shfl_up_sync(0xffffffffu, part, d); if (lane >= d) part += x; }
    all = __shfl_sync(0xffffffffu, part, SA_WARPS - 1);
    const u64 front = __shfl_sync(0xffffffffu, part, (warp + 31) & 31);
    return up - mine + (warp ? front : 0);
}
// descending; n: a power of two. A pair's sides 32 or fewer apart stay within a warp's places, so that stretches of steps need no block
__device__ __forceinline__ void sort_list(u64 * list, int n) {
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            for (int i = threadIdx.x; i < n / 2; i += SA_THREADS) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const u64 x = list[a], y = list[b];
                if ((x < y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
            }
            if (j > 32 || (j == 1 && k >= 64)) __syncthreads(); else __syncwarp();
        }
    __syncthreads();
}

// four neighbouring logits of the slice in shared memory
template <typename T> __device__ __forceinline__ void four_of(const T * vals, int g, float (&v)[4]) {
    const Four<T> f = reinterpret_cast<const Four<T> *>(vals)[g];
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = to_f(f.v[e]);
}

// floor(16 x logit), as the last bits of 1.5 x 2^23 + 16 x logit rounded down; logits beyond +-262143 stand with those, a NaN with -infinity
constexpr float SA_FAR = 262143.f;
__device__ __forceinline__ int bin_place(float v) { return __float_as_int(__fmaf_rd(fminf(fmaxf(v, -SA_FAR), SA_FAR), SA_PER_NAT, 12582912.f)) - 0x4b400000; }
// the smallest float whose place is p or more
__device__ __forceinline__ float place_from(int p) { return p <= (int) (-SA_FAR * SA_PER_NAT) ? -INFINITY : (float) p * (1.f / SA_PER_NAT); }

template <typename T>
__global__ void __launch_bounds__(SA_THREADS, 2) k_sample(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t sa_raw[];
    __shared__ SampleSmem sm;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int) cl.block_rank(), blocks = (int) cl.num_blocks();
    const int row = (int) (blockIdx.x / blocks), base = rank * a.slice, n = max(0, min(a.slice, a.n_vocab - base)), groups = (n + 3) >> 2;
    u64 * list = reinterpret_cast<u64 *>(sa_raw);                        // [SA_LIST]
    u64 * fine = list + SA_LIST;                                         // [SA_FINE] sums
    int * fine_count = reinterpret_cast<int *>(fine + SA_FINE), * bins = fine_count + SA_FINE;
    T * vals = reinterpret_cast<T *>(bins + SA_BINS);
    const float temperature = a.temperature ? a.temperature[row] : 1.f, top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f, u = a.u[row];
    const int k_all = a.top_k ? a.top_k[row] : 0, k = k_all > 0 && k_all < a.n_vocab ? k_all : 0;
    const bool by_p = top_p < 1.f, cut = temperature > 0.f && (k > 0 || by_p);
    int turn = 0;
    const auto add = [](u64 x, u64 y) { return x + y; };
    const auto each = [&](auto f) {                                      // f(four logits, index of the first in the slice)
        for (int g = tid; g < groups; g += SA_THREADS) { float v[4]; four_of(vals, g, v); f(v, 4 * g); }
    };
    // the slice, to whole fours, and its largest (a NaN is none)
    float top = -INFINITY;
    {
        const T * src = static_cast<const T *>(a.logits) + row * a.row_stride + base;
        constexpr int E = 16 / sizeof(T);
        for (int i = tid; i < SA_BINS; i += SA_THREADS) bins[i] = 0;
        if (tid < 16) sm.table[tid] = exp2((double) tid / 16.0);
        if (tid == 0) sm.n_list = 0;
        int done = 0;
        if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            done = n / E * E;
            for (int i0 = tid * E; i0 < done; i0 += 8 * SA_THREADS * E) {
                uint4 x[8];
#pragma unroll
                for (int j = 0; j < 8; j++) { const int i = i0 + j * SA_THREADS * E; if (i < done) x[j] = *reinterpret_cast<const uint4 *>(src + i); }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int i = i0 + j * SA_THREADS * E;
                    if (i < done) {
                        *reinterpret_cast<uint4 *>(vals + i) = x[j];
                        const Four<T> * f = reinterpret_cast<const Four<T> *>(&x[j]);
#pragma unroll
                        for (int h = 0; h < E / 4; h++)
#pragma unroll
                            for (int e = 0; e < 4; e++) top = fmaxf(top, to_f(f[h].v[e]));
                    }
                }
            }
        }
        for (int i = done + tid; i < 4 * groups; i += SA_THREADS) { const T x = i < n ? src[i] : from_f<T>(-INFINITY); vals[i] = x; top = fmaxf(top, to_f(x)); }
    }
    top = key_logit(warp_reduce(order_key(top, 0), [](u64 x, u64 y) { return max(x, y); }));
    if (lane == 0) sm.red[warp] = __float_as_uint(top);
    __syncthreads();
    for (int w = 0; w < SA_WARPS; w++) top = fmaxf(top, __uint_as_float((uint32_t) sm.red[w]));
    const int place = bin_place(top);
    if (tid == 0) { sm.top = top; sm.place = place; }
    if (cut)
        each([&](const float (&v)[4], int) {
#pragma unroll
            for (int e = 0; e < 4; e++) atomicAdd(&bins[min(SA_BINS - 1, place - bin_place(v[e]))], 1);
        });
    cl.sync();
    int places[SA_MAX_CLUSTER], row_place = (int) (-SA_FAR * SA_PER_NAT);
#pragma unroll
    for (int r = 0; r < SA_MAX_CLUSTER; r++) {
        const SampleSmem * o = cl.map_shared_rank(&sm, r < blocks ? r : 0);
        places[r] = o->place;
        row_place = max(row_place, places[r]);
        top = fmaxf(top, o->top);
    }
    const auto finish = [&](int id, float lp) { a.ids[row] = id; if (a.logprobs) a.logprobs[row] = lp; };
    const auto first_of_largest = [&]() {
        u64 mine = ~0ull;
        each([&](const float (&v)[4], int i) {
#pragma unroll
            for (int e = 3; e >= 0; e--) if (v[e] == top) mine = min(mine, (u64) (base + i + e));
        });
        return (int) cluster_join(cl, sm, mine, ~0ull, turn, [](u64 x, u64 y) { return min(x, y); });
    };
    if (top == -INFINITY || !(temperature > 0.f)) {                      // (behind the join nobody reads here any more)
        const int i = first_of_largest();
        if (rank == 0 && tid == 0) finish(top == -INFINITY ? -1 : i, top == -INFINITY ? -INFINITY : 0.f);
        return;
    }
    const auto exactly = [&](float v) { return v == top ? 0.0 : (double) top - (double) v; };   // how far a logit is from the largest
    // Weights are 0 from 28.5 (x temperature) below the largest on, so that the cut at 30, in floats, decides nothing. (An infinity as the largest: only others like it have a weight.)
    constexpr float MOST = 3.402823466e38f;
    const double cold = 1.0 / (double) temperature, steps = 1.0 / SA_LN, steps_cold = steps * cold, top_d = (double) fminf(top, MOST);
    const float from_1 = fmaxf((float) ((double) top - 30.0), -MOST), from_t = fmaxf((float) ((double) top - 30.0 * (double) temperature), -MOST);
    const auto weight = [&](float v) { return fixed_weight((double) fminf(v, MOST) - top_d, steps, v >= from_1, sm.table); };
    const auto tempered = [&](float v, bool in) { return fixed_weight((double) fminf(v, MOST) - top_d, steps_cold, in, sm.table); };
    // min-p keeps the logits from from_p on, the smallest float that is at most -log(min_p) below the largest (all where min_p is NaN, as top-p does)
    float from_p = -INFINITY;
    if (min_p > 0.f) {
        const double far = min_p < 1.f ? -log((double) min_p) : 0.0;
        from_p = fminf((float) ((double) top - far), top);
        for (int j = 0; j < 4 && exactly(from_p) > far; j++) from_p = nextafterf(from_p, INFINITY);
        for (int j = 0; j < 4 && exactly(nextafterf(from_p, -INFINITY)) <= far; j++) from_p = nextafterf(from_p, -INFINITY);
    }
    const auto log_share = [&](double x, u64 total) { return (float) (-(x == 0.0 ? 0.0 : x * cold) - log((double) total * (1.0 / SA_ONE))); };
    const auto target_of = [&](u64 total) { const double at = (double) u * (double) total; return at >= (double) total ? total - 1 : at > 0.0 ? (u64) at : 0; };
    u64 edge = 0;                                                        // tokens of keys >= edge are kept by top-k and top-p
    // the last key of the shortest prefix of the keys >= from that holds `want` tokens, or whose sum of weights reaches `want`
    const auto bisect = [&](u64 from, bool weights, double want) {
        u64 lo = from, hi = order_key(top, 0);                           // the prefix down to lo is enough
        while (lo < hi) {
            const u64 mid = lo + (hi - lo + 1) / 2;
            u64 mine = 0;
            each([&](const float (&v)[4], int i) {
#pragma unroll
                for (int e = 0; e < 4; e++) if (order_key(v[e], base + i + e) >= mid) mine += weights ? weight(v[e]) : i + e < n;
            });
            mine = cluster_join(cl, sm, mine, 0ull, turn, add);
            if ((double) mine >= want) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    // the tokens of logits lo to hi for which f holds, to the lists of the first `takers` blocks
    const auto gather = [&](int takers, float lo, float hi, auto f) {
        each([&](const float (&v)[4], int i) {
            bool in[4];
#pragma unroll
            for (int e = 0; e < 4; e++) in[e] = (v[e] >= lo) & (v[e] <= hi);
            if (!(in[0] | in[1] | in[2] | in[3])) return;
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (in[e] && f(v[e]) && i + e < n)
                    for (int r = 0; r < takers; r++) {
                        const int at = atomicAdd(&cl.map_shared_rank(&sm, r)->n_list, 1);
                        if (at < SA_LIST) cl.map_shared_rank(list, r)[at] = order_key(v[e], base + i + e);
                    }
        });
        cl.sync();
    };
    const auto sort_padded = [&](int m) {                                // the list in order, padded with zeros
        int pad = 32;
        while (pad < m) pad <<= 1;
        for (int i = m + tid; i < pad; i += SA_THREADS) list[i] = 0;
        __syncthreads();
        sort_list(list, pad);
    };
    if (cut) {
        // a bin of the row's a thread, over all blocks; what lies behind the last but one is the rest
        int cnt = 0, theirs[SA_MAX_CLUSTER];
#pragma unroll
        for (int r = 0; r < SA_MAX_CLUSTER; r++) theirs[r] = cl.map_shared_rank(bins, r < blocks ? r : 0)[max(tid - (row_place - places[r]), 0)];       // (a block's places are the row's or lower)
#pragma unroll
        for (int r = 0; r < SA_MAX_CLUSTER; r++) cnt += r < blocks && tid >= row_place - places[r] ? theirs[r] : 0;
        if (tid == SA_BINS - 1) cnt = 0;
        u64 counted;
        const u64 front = block_before64((u64) cnt, counted, sm.red);
        if (tid == SA_BINS - 1) cnt = a.n_vocab - (int) counted;
        if (tid == 0) { sm.answer[0] = 0; sm.answer[1] = SA_BINS - 1; sm.answer[2] = sm.answer[3] = 0; }
        __syncthreads();
        if (k > 0) {
            if (front < (u64) k && front + cnt >= (u64) k) { sm.answer[1] = tid; sm.answer[3] = front + cnt; }
        } else if (fabsf(top) < SA_FAR) {
            // A bin's tokens lie (b - 1) / 16 + s to b / 16 + s below the largest, s what the largest is above its bin's lower end: bounds of each bin's sum, widened by 1e-4 for the
            // roundings of either side. C, the sum up to a bin's end, has the share p when (1 - p) C >= p (what lies behind)
            const double s = (double) top - (double) row_place / SA_PER_NAT, p = (double) top_p, e = exp(-(double) tid / SA_PER_NAT - s) * SA_ONE * cnt;
            const u64 l = tid == SA_BINS - 1 ? 0 : (u64) (e * 0.9999), h = (u64) fmin(e * (1.064495 * 1.0001), SA_ONE * cnt) + cnt;      // exp(1 / 16); each token's weight is rounded by half a step
            u64 low_all, high_all;
            const u64 in_l = block_before64(l, low_all, sm.red), in_h = block_before64(h, high_all, sm.red);
            const auto surely = [&](u64 low, u64 high) { return (1.0 - p) * (double) low >= p * (double) (high_all - high); };
            const auto maybe = [&](u64 low, u64 high) { return (1.0 - p) * (double) high * 1.0001 >= p * (double) (low_all - low); };
            if (maybe(in_l + l, in_h + h) && (tid == 0 || !maybe(in_l, in_h))) { sm.answer[0] = tid; sm.answer[2] = front; }
            if (surely(in_l + l, in_h + h) && (tid == 0 || !surely(in_l, in_h))) { sm.answer[1] = tid; sm.answer[3] = front + cnt; }
        }
        __syncthreads();
        const int b_lo = (int) sm.answer[0], b_hi = (int) sm.answer[1];
        const float v_hi = b_lo ? place_from(row_place - b_lo + 1) : INFINITY, v_lo = b_hi == SA_BINS - 1 ? -INFINITY : place_from(row_place - b_hi);      // logits from v_lo to below v_hi
        if (k > 0 && sm.answer[3] <= SA_LIST) {
            // everything that can be kept: the first block ends the row
            gather(1, v_lo, INFINITY, [](float) { return true; });
            if (rank) return;
            const int m = sm.n_list;
            if (m <= SA_SHORT) {                                         // a thread a token, which goes through all of them twice
                u64 * w_of = fine, * t_of = fine + SA_SHORT;                 // (over the counts and the bins, which all blocks have read)
                static_assert(16 * SA_SHORT <= 12 * SA_FINE + 4 * SA_BINS, "two numbers a token");
                const u64 mine = tid < m ? list[tid] : 0, w = tid < m ? weight(key_logit(mine)) : 0;
                w_of[tid] = w;
                __syncthreads();
                int before_me = 0;
                u64 c = 0;
                if (tid < m)
#pragma unroll 4
                    for (int j = 0; j < m; j++) { const bool first = list[j] > mine; before_me += first; c += first ? w_of[j] : 0; }
                if (tid < m && before_me == min(k, m) - 1) sm.answer[0] = c + w;
                __syncthreads();
                const bool in = tid < m && before_me < k && (before_me == 0 || !by_p || (double) c < (double) top_p * (double) sm.answer[0]) && key_logit(mine) >= from_p;
                const u64 t = tempered(key_logit(mine), in && key_logit(mine) >= from_t);
                t_of[tid] = t;
                __syncthreads();
                if (in) {
                    u64 total = 0, upto = 0;
#pragma unroll 4
                    for (int j = 0; j < m; j++) { total += t_of[j]; upto += (uint32_t) list[j] >= (uint32_t) mine ? t_of[j] : 0; }       // (~index)
                    const u64 target = target_of(total);
                    if (upto - t <= target && target < upto) finish(key_index(mine), log_share(exactly(key_logit(mine)), total));
                }
                return;
            }
            const int per = (m + SA_THREADS - 1) / SA_THREADS, i0 = min(m, tid * per), i1 = min(m, i0 + per);
            sort_padded(m);
            u64 mine_w = 0, all, kept = 0;
            for (int i = i0; i < min(i1, k); i++) mine_w += weight(key_logit(list[i]));
            u64 c = block_before64(mine_w, all, sm.red);
            const double share = (double) top_p * (double) all;
            for (int i = i0; i < min(i1, k); i++) {                      // a token is kept while the sum in front of it is short of the share; the first always is
                const u64 w = weight(key_logit(list[i]));
                kept += (i == 0 || !by_p || (double) c < share) && (key_logit(list[i]) >= from_p);
                c += w;
            }
            block_before64(kept, all, sm.red);
            const int n_kept = (int) all;                                // a prefix
            // by index: what is kept, as (~index, logit)
            u64 swapped[SA_LIST / SA_THREADS];
#pragma unroll
            for (int j = 0; j < SA_LIST / SA_THREADS; j++) { const int i = tid + j * SA_THREADS; if (i < n_kept) { const u64 x = list[i]; swapped[j] = x << 32 | __float_as_uint(key_logit(x)); } }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < SA_LIST / SA_THREADS; j++) { const int i = tid + j * SA_THREADS; if (i < n_kept) list[i] = swapped[j]; }
            sort_padded(n_kept);
            const int d0 = min(n_kept, tid * per), d1 = min(n_kept, d0 + per);
            u64 sum = 0;
            for (int i = d0; i < d1; i++) { const float v = __uint_as_float((uint32_t) list[i]); sum += tempered(v, v >= from_t); }
            c = block_before64(sum, all, sm.red);
            const u64 target = target_of(all);
            if (c <= target && target < c + sum) {
                for (int i = d0; i < d1; i++) {
                    const float v = __uint_as_float((uint32_t) list[i]);
                    c += tempered(v, v >= from_t);
                    if (c > target) { finish((int) ~(uint32_t) (list[i] >> 32), log_share(exactly(v), all)); break; }
                }
            }
            return;
        }
        if (k > 0) {
            edge = bisect(0, false, (double) k);
            if (by_p) {
                u64 mine_w = 0;
                each([&](const float (&v)[4], int i) {
#pragma unroll
                    for (int e = 0; e < 4; e++) if (order_key(v[e], base + i + e) >= edge) mine_w += weight(v[e]);
                });
                const double share = (double) top_p * (double) cluster_join(cl, sm, mine_w, 0ull, turn, add);
                edge = share > 0.0 ? bisect(edge, true, share) : order_key(top, first_of_largest());
            }
        } else {
            // all weights, those in front of the bins, and those in the bins by finer ones
            const float from = b_lo ? v_hi : top, by = SA_FINE * SA_PER_NAT / (float) (b_hi - b_lo + 1);
            const auto fine_place = [&](float v) { return fminf((from - v) * by, (float) (SA_FINE - 1)); };       // its whole part is the finer bin
            const auto between = [&](float v) { return (v >= v_lo) & (v < v_hi); };
            for (int i = tid; i < SA_FINE; i += SA_THREADS) { fine[i] = 0; fine_count[i] = 0; }
            __syncthreads();
            u64 all = 0, in_front = 0;
            each([&](const float (&v)[4], int i) {
                u64 w[4];
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] = weight(v[e]);
                all += w[0] + w[1] + (w[2] + w[3]);
#pragma unroll
                for (int e = 0; e < 4; e++) in_front += v[e] >= v_hi ? w[e] : 0;
                if (!(between(v[0]) | between(v[1]) | between(v[2]) | between(v[3]))) return;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (between(v[e]) & (i + e < n)) {
                        const int b = (int) fine_place(v[e]);
                        atomicAdd(&fine[b], w[e]);
                        atomicAdd(&fine_count[b], 1);
                    }
            });
            u64 sums[2];
            block_before64(all, sums[0], sm.red);
            block_before64(in_front, sums[1], sm.red);
            if (tid < blocks) { cl.map_shared_rank(&sm, tid)->sums[rank][0] = sums[0]; cl.map_shared_rank(&sm, tid)->sums[rank][1] = sums[1]; }
            cl.sync();
            all = in_front = 0;
            for (int r = 0; r < blocks; r++) { all += sm.sums[r][0]; in_front += sm.sums[r][1]; }
            const double want = (double) top_p * (double) all;
            u64 w = 0, x[SA_MAX_CLUSTER];
            int fc = 0, y[SA_MAX_CLUSTER];
#pragma unroll
            for (int r = 0; r < SA_MAX_CLUSTER; r++) { const int o = r < blocks ? r : 0; x[r] = cl.map_shared_rank(fine, o)[tid]; y[r] = cl.map_shared_rank(fine_count, o)[tid]; }
#pragma unroll
            for (int r = 0; r < SA_MAX_CLUSTER; r++) if (r < blocks) { w += x[r]; fc += y[r]; }
            u64 c = in_front + block_before64(w, counted, sm.red);
            if (tid == 0) sm.answer[0] = SA_FINE;
            __syncthreads();
            if ((double) c < want && (double) (c + w) >= want) { sm.answer[0] = tid; sm.answer[1] = c; sm.answer[2] = fc; }
            __syncthreads();
            const int f_bin = (int) sm.answer[0];
            c = sm.answer[1];
            if (f_bin < SA_FINE && sm.answer[2] <= SA_LIST) {
                // bounds of the bin's logits, widened by far more than fine_place rounds, in front of the test itself
                const float slack = 1e-5f * (fabsf(from) + SA_FINE / by), f_lo = from - (float) (f_bin + 1) / by - slack, f_hi = from - (float) f_bin / by + slack;
                gather(blocks, f_bin == SA_FINE - 1 ? -INFINITY : f_lo, f_hi, [&](float v) { const float at = fine_place(v); return between(v) & (at >= (float) f_bin) & (at < (float) (f_bin + 1)); });
                const int m = sm.n_list;
                if (m <= SA_SHORT) {
                    const u64 mine = tid < m ? list[tid] : 0, w_mine = tid < m ? weight(key_logit(mine)) : 0;
                    if (tid == 0) sm.answer[0] = 0;
                    fine[tid] = w_mine;                                  // (everybody has read the sums)
                    __syncthreads();
                    if (tid < m) {
#pragma unroll 4
                        for (int j = 0; j < m; j++) c += list[j] > mine ? fine[j] : 0;
                        if ((double) c < want && (double) (c + w_mine) >= want) sm.answer[0] = mine;
                    }
                } else {
                    const int per = (m + SA_THREADS - 1) / SA_THREADS, i0 = min(m, tid * per), i1 = min(m, i0 + per);
                    sort_padded(m);
                    u64 mine_w = 0;
                    for (int i = i0; i < i1; i++) mine_w += weight(key_logit(list[i]));
                    c += block_before64(mine_w, counted, sm.red);
                    if (tid == 0) sm.answer[0] = 0;
                    __syncthreads();
                    for (int i = i0; i < i1; i++) {
                        const u64 w_i = weight(key_logit(list[i]));
                        if ((double) c < want && (double) (c + w_i) >= want) sm.answer[0] = list[i];
                        c += w_i;
                    }
                }
                __syncthreads();
                edge = sm.answer[0];
            } else edge = want > 0.0 ? bisect(0, true, want) : order_key(top, first_of_largest());
        }
    }
    // the draw: sums of 128 neighbouring tokens, a warp's at a time, which stand in order of index
    const float edge_logit = edge ? key_logit(edge) : -INFINITY, from = fmaxf(fmaxf(from_t, from_p), edge_logit);
    const int edge_index = edge ? key_index(edge) : 0x7fffffff;
    const auto drawn = [&](const float (&v)[4], int i, u64 (&w)[4]) {
        bool in[4];
#pragma unroll
        for (int e = 0; e < 4; e++) { in[e] = v[e] >= from; w[e] = 0; }
        if (!(in[0] | in[1] | in[2] | in[3])) return;
        if ((v[0] == edge_logit) | (v[1] == edge_logit) | (v[2] == edge_logit) | (v[3] == edge_logit))
#pragma unroll
            for (int e = 0; e < 4; e++) in[e] = in[e] & ((v[e] != edge_logit) | (base + i + e <= edge_index));
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = tempered(v[e], in[e]);
    };
    const int sweeps = (groups + SA_THREADS - 1) / SA_THREADS;
    for (int s = 0; s < sweeps; s++) {
        const int g = s * SA_THREADS + tid;
        u64 sum = 0;
        if (g < groups) {
            float v[4];
            u64 w[4];
            four_of(vals, g, v);
            drawn(v, 4 * g, w);
            sum = w[0] + w[1] + w[2] + w[3];
        }
        if (__any_sync(0xffffffffu, sum != 0)) sum = warp_sum(sum);
        if (lane == 0) sm.parts[s][warp] = sum;
    }
    __syncthreads();
    u64 mine = tid < sweeps * SA_WARPS ? sm.parts[tid / SA_WARPS][tid % SA_WARPS] : 0, block_sum;      // (256 parts at most)
    const u64 in_block = block_before64(mine, block_sum, sm.red);
    if (tid < blocks) cl.map_shared_rank(&sm, tid)->each[rank] = block_sum;
    cl.sync();
    u64 total = 0, front = in_block;
    for (int r = 0; r < blocks; r++) { if (r < rank) front += sm.each[r]; total += sm.each[r]; }
    const u64 target = target_of(total);
    if (tid == 0) sm.answer[3] = ~0ull;
    __syncthreads();
    if (front <= target && target < front + mine) { sm.answer[2] = front; sm.answer[3] = tid; }        // one part of the cluster
    __syncthreads();
    if (warp == 0 && sm.answer[3] != ~0ull) {
        const int at = (int) sm.answer[3], g = at / SA_WARPS * SA_THREADS + at % SA_WARPS * 32 + lane;
        float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (g < groups) four_of(vals, g, v);
        u64 w[4], sum = 0;
        drawn(v, 4 * g, w);
        sum = w[0] + w[1] + w[2] + w[3];
        u64 up = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const u64 x = __shfl_up_sync(0xffffffffu, up, d); if (lane >= d) up += x; }
        u64 c = sm.answer[2] + up - sum;
        if (c <= target && target < c + sum)
            for (int e = 0; e < 4; e++) {
                c += w[e];
                if (c > target) { finish(base + 4 * g + e, log_share(exactly(v[e]), total)); break; }
            }
    }
}

}  // namespace srv
}  // namespace b200
