// serve_sample.cuh — the draw of next tokens from rows of logits (sm_100a).
//
// A row's tokens are ordered by logit, the lower index first among equals. Each filter keeps a prefix of that order: top-k the first k; top-p, of those, the shortest prefix with at least
// the share p of their weight exp(logit - largest); min-p those of weight at least min_p. Of what all three keep, token i is drawn with weight exp((logit - largest) / temperature): the
// first one in order of index at which the sum exceeds u x total. A filter's edge and the draw are decisions on sums, so weights are whole multiples of 2^-40 from 64-bit exponentials and
// sums of them are exact: no order of summation, and no other split of the row, changes a result.
//
// A cluster of blocks takes a row and holds its slice in shared memory: logits cross HBM once. One sweep finds the maximum. A histogram of (largest - logit) by 1 / 32 gives, from counts
// alone, the bin of the k-th token, and bounds between which the sum for top-p is crossed; only tokens of those bins are sorted (a few hundred of 128 k), exactly as the definition says.
// With top-k all that can be kept is in that list, and the first block ends the row by itself. Otherwise a last sweep sums what is kept, 128 tokens at a time, and the warp in whose tokens
// the draw falls looks for it. Rows whose edge lies among more than 2048 candidates (thousands of equal logits, very large k) are bisected over (logit, index) instead.
#pragma once
#include "serve_cache.cuh"
#include <cooperative_groups.h>

namespace b200 {
namespace srv {

namespace cg = cooperative_groups;

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32, SA_BINS = 1024, SA_LIST = 2048, SA_MAX_CLUSTER = 8, SA_MAX_VOCAB = 1 << 18, SA_SWEEPS = SA_MAX_VOCAB / SA_MAX_CLUSTER / SA_THREADS / 4;
constexpr float SA_PER_NAT = 32.f;
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

// 2^40 exp(-x) to the nearest whole number, x >= 0: 2^n times the series of e^f, |f| <= ln 2 / 2, whose first term left out is below 2^-46
__device__ __forceinline__ u64 fixed_weight(double x) {
    if (!(x < 30.0)) return 0;
    const double y = x * -1.4426950408889634, n = rint(y), f = (y - n) * 0.6931471805599453;
    double p = 1.0 / 479001600.0;
    p = fma(p, f, 1.0 / 39916800.0);
    p = fma(p, f, 1.0 / 3628800.0);
    p = fma(p, f, 1.0 / 362880.0);
    p = fma(p, f, 1.0 / 40320.0);
    p = fma(p, f, 1.0 / 5040.0);
    p = fma(p, f, 1.0 / 720.0);
    p = fma(p, f, 1.0 / 120.0);
    p = fma(p, f, 1.0 / 24.0);
    p = fma(p, f, 1.0 / 6.0);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return (u64) __double2ull_rn(p * __longlong_as_double((long long) (1023 + 40 + (int) n) << 52));
}

// (logit, index) as one number: larger is earlier in the order
__device__ __forceinline__ u64 order_key(float v, int i) {
    const uint32_t b = __float_as_uint(v);
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
struct SampleSmem {
    u64 red[SA_WARPS], each[SA_MAX_CLUSTER], turn[2][SA_MAX_CLUSTER];
    u64 answer[4], edge;
    u64 parts[SA_SWEEPS][SA_WARPS];
    int n_list;
};
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

template <typename T>
__global__ void __launch_bounds__(SA_THREADS, 2) k_sample(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t sa_raw[];
    __shared__ SampleSmem sm;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int) cl.block_rank(), blocks = (int) cl.num_blocks();
    const int row = (int) (blockIdx.x / blocks), base = rank * a.slice, n = max(0, min(a.slice, a.n_vocab - base)), groups = (n + 3) >> 2;
    u64 * list = reinterpret_cast<u64 *>(sa_raw);                        // [SA_LIST]; before it is a list, [SA_BINS] fine sums and counts
    int * bins = reinterpret_cast<int *>(sa_raw + 8 * SA_LIST);          // [SA_BINS]
    T * vals = reinterpret_cast<T *>(sa_raw + 8 * SA_LIST + 4 * SA_BINS);
    int turn = 0;
    // the slice, to whole fours
    {
        const T * src = static_cast<const T *>(a.logits) + row * a.row_stride + base;
        constexpr int E = 16 / sizeof(T);
        int done = 0;
        if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            done = n / E * E;
            for (int i = tid * E; i < done; i += SA_THREADS * E)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"((uint32_t) __cvta_generic_to_shared(vals + i)), "l"(src + i) : "memory");
        }
        for (int i = done + tid; i < 4 * groups; i += SA_THREADS) vals[i] = i < n ? src[i] : from_f<T>(-INFINITY);
        for (int i = tid; i < SA_BINS; i += SA_THREADS) bins[i] = 0;
        if (tid == 0) sm.n_list = 0;
    }
    const float temperature = a.temperature ? a.temperature[row] : 1.f, top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? fminf(a.min_p[row], 1.f) : 0.f;
    const int k_all = a.top_k ? a.top_k[row] : 0, k = k_all > 0 && k_all < a.n_vocab ? k_all : 0;
    const float u = a.u[row];
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    const auto add = [](u64 x, u64 y) { return x + y; };
    // the largest; a NaN becomes -infinity and -0 becomes 0 on the way
    float top = -INFINITY;
    for (int g = tid; g < groups; g += SA_THREADS) {
        float v[4];
        four_of(vals, g, v);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (v[e] != v[e] || __float_as_uint(v[e]) == 0x80000000u) { v[e] = v[e] == 0.f ? 0.f : -INFINITY; vals[4 * g + e] = from_f<T>(v[e]); }
            top = fmaxf(top, v[e]);
        }
    }
    top = key_logit(cluster_join(cl, sm, order_key(top, 0), 0ull, turn, [](u64 x, u64 y) { return max(x, y); }));
    const auto finish = [&](int id, float lp) { a.ids[row] = id; if (a.logprobs) a.logprobs[row] = lp; };
    const auto each = [&](auto f) {                                      // f(four logits, index of the first in the slice)
        for (int g = tid; g < groups; g += SA_THREADS) { float v[4]; four_of(vals, g, v); f(v, 4 * g); }
    };
    const auto first_of_largest = [&]() {
        u64 mine = ~0ull;
        each([&](const float (&v)[4], int i) {
#pragma unroll
            for (int e = 3; e >= 0; e--) if (v[e] == top) mine = min(mine, (u64) (base + i + e));
        });
        return (int) cluster_join(cl, sm, mine, ~0ull, turn, [](u64 x, u64 y) { return min(x, y); });
    };
    if (top == -INFINITY || !(temperature > 0.f)) {
        const int i = top == -INFINITY ? -1 : first_of_largest();
        if (rank == 0 && tid == 0) finish(i, i < 0 ? -INFINITY : 0.f);
        return;                                                          // (the join was the last that others read here)
    }
    const auto below = [&](float v) { return v == top ? 0.f : top - v; };                       // how far a logit is from the largest, to a float
    const auto exactly = [&](float v) { return v == top ? 0.0 : (double) top - (double) v; };
    const auto weight = [&](float v) { return fixed_weight(exactly(v)); };
    const auto bin_of = [&](float v) { return (int) fminf(below(v) * SA_PER_NAT, (float) (SA_BINS - 1)); };
    const float far = min_p > 0.f ? 0.01f - logf(min_p) : INFINITY;      // nothing so far below the largest is kept by min-p
    const double cold = 1.0 / (double) temperature;
    const auto tempered = [&](double x) { return fixed_weight(x == 0.0 ? 0.0 : x * cold); };
    const auto log_share = [&](double x, u64 total) { return (float) (-(x == 0.0 ? 0.0 : x * cold) - log((double) total * (1.0 / SA_ONE))); };
    const auto target_of = [&](u64 total) { const double at = (double) u * (double) total; return at >= (double) total ? total - 1 : at > 0.0 ? (u64) at : 0; };
    u64 edge = 0;                                                        // tokens of keys >= edge are kept by top-k and top-p
    const bool by_p = top_p < 1.f;
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
    // list of the tokens for which f holds, in the first block of the cluster
    const auto gather = [&](auto f) {
        SampleSmem * s0 = cl.map_shared_rank(&sm, 0);
        u64 * l0 = cl.map_shared_rank(list, 0);
        each([&](const float (&v)[4], int i) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (f(v[e]) && i + e < n) {
                    const int at = atomicAdd(&s0->n_list, 1);
                    if (at < SA_LIST) l0[at] = order_key(v[e], base + i + e);
                }
        });
        cl.sync();
    };
    const auto sort_padded = [&](int m) {                                // first block: the list in order, padded with zeros
        int pad = 32;
        while (pad < m) pad <<= 1;
        for (int i = m + tid; i < pad; i += SA_THREADS) list[i] = 0;
        __syncthreads();
        sort_list(list, pad);
    };
    if (k > 0 || by_p) {
        u64 total = 0, mine = 0;
        each([&](const float (&v)[4], int i) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (i + e < n) atomicAdd(&bins[bin_of(v[e])], 1);
                if (k == 0) mine += weight(v[e]);
            }
        });
        if (k == 0) total = cluster_join(cl, sm, mine, 0ull, turn, add);
        else cl.sync();
        // two bins a thread, over all blocks
        int cnt[2] = {0, 0};
        for (int r = 0; r < blocks; r++) {
            const int2 v = reinterpret_cast<const int2 *>(cl.map_shared_rank(bins, r))[tid];
            cnt[0] += v.x; cnt[1] += v.y;
        }
        u64 dummy;
        const u64 front = block_before64((u64) (cnt[0] + cnt[1]), dummy, sm.red);
        if (tid == 0) { sm.answer[0] = 0; sm.answer[1] = SA_BINS - 1; sm.answer[2] = sm.answer[3] = 0; }
        __syncthreads();
        const double want = (double) top_p * (double) total;
        if (k > 0) {
            u64 c = front;
            for (int j = 0; j < 2; j++) {
                if (c < (u64) k && c + cnt[j] >= (u64) k) { sm.answer[1] = 2 * tid + j; sm.answer[3] = c + cnt[j]; }
                c += cnt[j];
            }
        } else {
            // a bin's sum lies between cnt exp(-(b + 1) / 32) and cnt exp(-b / 32), widened by 1e-4 for the roundings of either side. The sum up to a bin's end is bounded by the bins in
            // front and, from the exact total, by those behind, which is the sharper of the two near the end
            u64 low = 0, high = 0, l[2], h[2], low_all, high_all;
            for (int j = 0; j < 2; j++) {
                const double e = exp(-(double) (2 * tid + j) / SA_PER_NAT) * SA_ONE;
                h[j] = (u64) (cnt[j] * e * 1.0001); l[j] = 2 * tid + j == SA_BINS - 1 ? 0 : (u64) (cnt[j] * e * 0.96923 * 0.9999);
                low += l[j]; high += h[j];
            }
            u64 cl_ = block_before64(low, low_all, sm.red), ch = block_before64(high, high_all, sm.red);
            const auto least = [&](u64 in_l, u64 in_h) { return fmax((double) in_l, (double) total - (double) (high_all - in_h)); };
            const auto most = [&](u64 in_l, u64 in_h) { return fmin((double) in_h, (double) total - (double) (low_all - in_l)); };
            u64 c = front;
            for (int j = 0; j < 2; j++) {
                if (most(cl_, ch) < want && most(cl_ + l[j], ch + h[j]) >= want) { sm.answer[0] = 2 * tid + j; sm.answer[2] = c; }
                if (least(cl_, ch) < want && least(cl_ + l[j], ch + h[j]) >= want) sm.answer[1] = 2 * tid + j;
                c += cnt[j]; cl_ += l[j]; ch += h[j];
            }
            __syncthreads();
            c = front;
            for (int j = 0; j < 2; j++) { c += cnt[j]; if (2 * tid + j == (int) sm.answer[1]) sm.answer[3] = c; }
        }
        __syncthreads();
        const int b_lo = (int) sm.answer[0], b_hi = (int) sm.answer[1];
        int n_between = (int) (sm.answer[3] - sm.answer[2]);
        if (k > 0 && n_between <= SA_LIST) {
            // everything that can be kept: the first block ends the row
            gather([&](float v) { return bin_of(v) <= b_hi; });
            if (rank) return;
            const int m = sm.n_list, per = (m + SA_THREADS - 1) / SA_THREADS, i0 = min(m, tid * per), i1 = min(m, i0 + per);
            sort_padded(m);
            u64 mine_w = 0, all, kept = 0;
            for (int i = i0; i < min(i1, k); i++) mine_w += weight(key_logit(list[i]));
            u64 c = block_before64(mine_w, all, sm.red);
            const double share = (double) top_p * (double) all;
            for (int i = i0; i < min(i1, k); i++) {                      // a token is kept while the sum in front of it is short of the share; the first always is
                const u64 w = weight(key_logit(list[i]));
                kept += (i == 0 || !by_p || (double) c < share) && !((double) w < (double) min_p * SA_ONE);
                c += w;
            }
            int n_kept;
            block_before64(kept, all, sm.red);
            n_kept = (int) all;                                          // a prefix
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
            for (int i = d0; i < d1; i++) sum += tempered(exactly(__uint_as_float((uint32_t) list[i])));
            c = block_before64(sum, all, sm.red);
            const u64 target = target_of(all);
            if (c <= target && target < c + sum) {
                for (int i = d0; i < d1; i++) {
                    const double x = exactly(__uint_as_float((uint32_t) list[i]));
                    c += tempered(x);
                    if (c > target) { finish((int) ~(uint32_t) (list[i] >> 32), log_share(x, all)); break; }
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
            u64 in_front = 0;                                            // sum of the bins in front of b_lo
            each([&](const float (&v)[4], int) {
#pragma unroll
                for (int e = 0; e < 4; e++) if (bin_of(v[e]) < b_lo) in_front += weight(v[e]);
            });
            in_front = cluster_join(cl, sm, in_front, 0ull, turn, add);
            const float f_lo = (float) b_lo / SA_PER_NAT, f_scale = SA_BINS * SA_PER_NAT / (float) (b_hi - b_lo + 1);
            const auto fine_bin = [&](float v) { return (int) fminf((below(v) - f_lo) * f_scale, (float) (SA_BINS - 1)); };
            int f_bin = -1;
            if (n_between > SA_LIST) {                                   // 1024 finer bins between b_lo and b_hi, their sums exact
                u64 * fine = list;
                int * count = reinterpret_cast<int *>(fine + SA_BINS);
                for (int i = tid; i < SA_BINS; i += SA_THREADS) { fine[i] = 0; count[i] = 0; }
                __syncthreads();
                each([&](const float (&v)[4], int i) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int b = bin_of(v[e]);
                        if (b >= b_lo && b <= b_hi && i + e < n) {
                            atomicAdd(&fine[fine_bin(v[e])], weight(v[e]));
                            atomicAdd(&count[fine_bin(v[e])], 1);
                        }
                    }
                });
                cl.sync();
                u64 w[2] = {0, 0};
                int fc[2] = {0, 0};
                for (int r = 0; r < blocks; r++) {
                    const u64 * fw = cl.map_shared_rank(fine, r) + 2 * tid;
                    const int * ff = cl.map_shared_rank(count, r) + 2 * tid;
                    for (int j = 0; j < 2; j++) { w[j] += fw[j]; fc[j] += ff[j]; }
                }
                u64 c = in_front + block_before64(w[0] + w[1], dummy, sm.red);
                if (tid == 0) sm.answer[0] = SA_BINS;
                __syncthreads();
                for (int j = 0; j < 2; j++) {
                    if ((double) c < want && (double) (c + w[j]) >= want) { sm.answer[0] = 2 * tid + j; sm.answer[1] = c; sm.answer[2] = fc[j]; }
                    c += w[j];
                }
                __syncthreads();
                if (sm.answer[0] < SA_BINS) { f_bin = (int) sm.answer[0]; in_front = sm.answer[1]; n_between = (int) sm.answer[2]; }
                cl.sync();                                               // the sums have been read: a list may take their place
            }
            if (n_between <= SA_LIST) {
                gather([&](float v) {
                    const int b = bin_of(v);
                    return b >= b_lo && b <= b_hi && (f_bin < 0 || fine_bin(v) == f_bin);
                });
                if (rank == 0) {
                    const int m = sm.n_list, per = (m + SA_THREADS - 1) / SA_THREADS, i0 = min(m, tid * per), i1 = min(m, i0 + per);
                    sort_padded(m);
                    u64 mine_w = 0, all;
                    for (int i = i0; i < i1; i++) mine_w += weight(key_logit(list[i]));
                    u64 c = in_front + block_before64(mine_w, all, sm.red);
                    if (tid == 0) sm.answer[0] = m ? list[m - 1] : 0;
                    __syncthreads();
                    for (int i = i0; i < i1; i++) {
                        const u64 w = weight(key_logit(list[i]));
                        if ((i == 0 || (double) c < want) && (double) (c + w) >= want) sm.answer[0] = list[i];
                        c += w;
                    }
                    __syncthreads();
                    const u64 e = sm.answer[0];
                    if (tid < blocks) cl.map_shared_rank(&sm, tid)->edge = e;
                }
                cl.sync();
                edge = sm.edge;
            } else edge = want > 0.0 ? bisect(0, true, want) : order_key(top, first_of_largest());
        }
    }
    // the draw: sums of 128 neighbouring tokens, a warp's at a time, which stand in order of index
    const auto drawn = [&](float v, int i) -> u64 {
        if (below(v) > far || v == -INFINITY || (edge && order_key(v, base + i) < edge)) return 0;
        const double x = exactly(v);
        if (min_p > 0.f && (double) fixed_weight(x) < (double) min_p * SA_ONE) return 0;
        return tempered(x);
    };
    const int sweeps = (groups + SA_THREADS - 1) / SA_THREADS;
    for (int s = 0; s < sweeps; s++) {
        const int g = s * SA_THREADS + tid;
        u64 sum = 0;
        if (g < groups) {
            float v[4];
            four_of(vals, g, v);
#pragma unroll
            for (int e = 0; e < 4; e++) sum += drawn(v[e], 4 * g + e);
        }
        if (__any_sync(0xffffffffu, sum != 0)) sum = warp_reduce(sum, add);
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
#pragma unroll
        for (int e = 0; e < 4; e++) { w[e] = drawn(v[e], 4 * g + e); sum += w[e]; }
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
