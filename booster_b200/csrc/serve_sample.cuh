// serve_sample.cuh — the draw of next tokens from rows of logits (sm_100a).
//
// A row's tokens are ordered by logit, the lower index first among equals. Each filter keeps a prefix of that order: top-k the first k; top-p, of those, the shortest prefix with at least
// the share p of their weight exp(logit - largest); min-p those of weight at least min_p. Of what all three keep, token i is drawn with weight exp((logit - largest) / temperature): the
// first one in order of index at which the sum exceeds u x total. A filter's edge and the draw are decisions on sums, so weights are whole multiples of 2^-40 from 64-bit exponentials and
// sums of them are exact: no order of summation, and no other split of the row, changes a result.
//
// A cluster of blocks takes a row and holds its slice in shared memory: logits cross HBM once. One pass finds the maximum. A histogram of (largest - logit) by 1 / 64 gives, from counts
// alone, the bin of the k-th token, and bounds between which the sum for top-p is crossed; only tokens of those bins are sorted (a few hundred of 128 k), exactly as the definition says.
// Rows whose edge lies among more than 4096 candidates (thousands of equal logits, very large k) are bisected over (logit, index) instead.
#pragma once
#include "serve_cache.cuh"
#include <cooperative_groups.h>

namespace b200 {
namespace srv {

namespace cg = cooperative_groups;

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32, SA_BINS = 2048, SA_LIST = 4096, SA_MAX_CLUSTER = 8;
constexpr float SA_PER_NAT = 64.f;
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
    u64 off = 0, sum = 0;
    for (int w = 0; w < SA_WARPS; w++) { if (w < warp) off += red[w]; sum += red[w]; }
    all = sum;
    return off + up - mine;
}
// descending
__device__ __forceinline__ void sort_list(u64 * list, int n) {        // n: a power of two
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            for (int i = threadIdx.x; i < n / 2; i += SA_THREADS) {
                const int a = 2 * i - (i & (j - 1)), b = a + j;
                const u64 x = list[a], y = list[b];
                if ((x < y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
            }
            __syncthreads();
        }
}

template <typename T>
__global__ void __launch_bounds__(SA_THREADS) k_sample(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t sa_raw[];
    __shared__ SampleSmem sm;
    cg::cluster_group cl = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int) cl.block_rank(), blocks = (int) cl.num_blocks();
    const int row = (int) (blockIdx.x / blocks), base = rank * a.slice, n = max(0, min(a.slice, a.n_vocab - base));
    u64 * list = reinterpret_cast<u64 *>(sa_raw);                        // [SA_LIST]; before it is a list: bins
    int * bins = reinterpret_cast<int *>(sa_raw);                        // [SA_BINS]
    u64 * fine = reinterpret_cast<u64 *>(sa_raw + 4 * SA_BINS);          // [SA_BINS] weights, then [SA_BINS] counts
    T * vals = reinterpret_cast<T *>(sa_raw + 8 * SA_LIST);
    const float temperature = a.temperature ? a.temperature[row] : 1.f, top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? fminf(a.min_p[row], 1.f) : 0.f;
    const int k_all = a.top_k ? a.top_k[row] : 0, k = k_all > 0 && k_all < a.n_vocab ? k_all : 0;
    int turn = 0;
    // the slice, and the first of the largest
    u64 first = 0;
    {
        const T * src = static_cast<const T *>(a.logits) + row * a.row_stride + base;
        constexpr int E = 16 / sizeof(T);
        int done = 0;
        if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
            done = n / E * E;
            for (int i = tid * E; i < done; i += SA_THREADS * E) *reinterpret_cast<uint4 *>(vals + i) = *reinterpret_cast<const uint4 *>(src + i);
        }
        for (int i = done + tid; i < n; i += SA_THREADS) vals[i] = src[i];
        for (int i = tid; i < SA_BINS; i += SA_THREADS) bins[i] = 0;
        if (tid == 0) sm.n_list = 0;
        __syncthreads();
    }
    const auto logit = [&](int i) { const float v = to_f(vals[i]) + 0.f; return v == v ? v : -INFINITY; };
    for (int i = tid; i < n; i += SA_THREADS) first = max(first, order_key(logit(i), base + i));
    first = cluster_join(cl, sm, first, 0ull, turn, [](u64 x, u64 y) { return max(x, y); });
    const float top = key_logit(first);
    const auto finish = [&](int id, float lp) { a.ids[row] = id; if (a.logprobs) a.logprobs[row] = lp; };
    if (top == -INFINITY || !(temperature > 0.f)) {
        if (rank == 0 && tid == 0) finish(top == -INFINITY ? -1 : key_index(first), top == -INFINITY ? -INFINITY : 0.f);
        cl.sync();
        return;
    }
    const auto below = [&](float v) { return v == top ? 0.f : top - v; };                       // how far a logit is from the largest, to a float
    const auto exactly = [&](float v) { return v == top ? 0.0 : (double) top - (double) v; };
    const auto weight = [&](float v) { return fixed_weight(exactly(v)); };
    const auto bin_of = [&](float v) { return (int) fminf(below(v) * SA_PER_NAT, (float) (SA_BINS - 1)); };
    const auto add = [](u64 x, u64 y) { return x + y; };
    const float far = min_p > 0.f ? 0.01f - logf(min_p) : INFINITY;     // nothing so far below the largest is kept by min-p
    u64 edge = 0;                                                        // tokens of keys >= edge are kept by top-k and top-p
    const bool by_p = top_p < 1.f;
    // the last key of the shortest prefix of the keys >= from that holds `want` tokens, or whose sum of weights reaches `want`
    const auto bisect = [&](u64 from, bool weights, double want) {
        u64 lo = from, hi = first;                                       // the prefix down to lo is enough
        while (lo < hi) {
            const u64 mid = lo + (hi - lo + 1) / 2;
            u64 mine = 0;
            for (int i = tid; i < n; i += SA_THREADS) {
                const float v = logit(i);
                if (order_key(v, base + i) >= mid) mine += weights ? weight(v) : 1;
            }
            mine = cluster_join(cl, sm, mine, 0ull, turn, add);
            if ((double) mine >= want) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    const auto sum_from = [&](u64 from) {
        u64 mine = 0;
        for (int i = tid; i < n; i += SA_THREADS) { const float v = logit(i); if (order_key(v, base + i) >= from) mine += weight(v); }
        return cluster_join(cl, sm, mine, 0ull, turn, add);
    };
    // list of the tokens whose f(bin, logit) holds, in the first block of the cluster
    const auto gather = [&](auto f) {
        for (int i = tid; i < n; i += SA_THREADS) {
            const float v = logit(i);
            if (f(v)) {
                SampleSmem * s0 = cl.map_shared_rank(&sm, 0);
                const int at = atomicAdd(&s0->n_list, 1);
                if (at < SA_LIST) cl.map_shared_rank(list, 0)[at] = order_key(v, base + i);
            }
        }
        cl.sync();
    };
    const auto sorted = [&]() {                                          // first block: the list in order, padded with zeros
        const int m = sm.n_list;
        int pad = 32;
        while (pad < m) pad <<= 1;
        for (int i = m + tid; i < pad; i += SA_THREADS) list[i] = 0;
        __syncthreads();
        sort_list(list, pad);
        return m;
    };
    if (k > 0 || by_p) {
        u64 total = 0, mine = 0;
        for (int i = tid; i < n; i += SA_THREADS) {
            const float v = logit(i);
            atomicAdd(&bins[bin_of(v)], 1);
            if (k == 0) mine += weight(v);
        }
        if (k == 0) total = cluster_join(cl, sm, mine, 0ull, turn, add);
        else cl.sync();
        // four bins a thread, over all blocks
        int cnt[4] = {0, 0, 0, 0};
        for (int r = 0; r < blocks; r++) {
            const int4 v = reinterpret_cast<const int4 *>(cl.map_shared_rank(bins, r))[tid];
            cnt[0] += v.x; cnt[1] += v.y; cnt[2] += v.z; cnt[3] += v.w;
        }
        int b_lo = 0, b_hi = SA_BINS - 1;
        u64 dummy;
        const u64 front = block_before64((u64) (cnt[0] + cnt[1] + cnt[2] + cnt[3]), dummy, sm.red);
        if (tid == 0) { sm.answer[0] = 0; sm.answer[1] = SA_BINS - 1; sm.answer[2] = sm.answer[3] = 0; }
        __syncthreads();
        if (k > 0) {
            u64 c = front;
            for (int j = 0; j < 4; j++) {
                if (c < (u64) k && c + cnt[j] >= (u64) k) { sm.answer[1] = 4 * tid + j; sm.answer[3] = c + cnt[j]; }
                c += cnt[j];
            }
        } else {
            // a bin's sum lies between cnt exp(-(b + 1) / 64) and cnt exp(-b / 64), widened by 1e-4 for the roundings of either side. The sum up to a bin's end is bounded by the bins in
            // front and, from the exact total, by those behind, which is the sharper of the two near the end
            const double want = (double) top_p * (double) total;
            u64 low = 0, high = 0, l[4], h[4], low_all, high_all;
            for (int j = 0; j < 4; j++) {
                const double e = exp(-(double) (4 * tid + j) / SA_PER_NAT) * 1099511627776.0;
                h[j] = (u64) (cnt[j] * e * 1.0001); l[j] = 4 * tid + j == SA_BINS - 1 ? 0 : (u64) (cnt[j] * e * 0.98449 * 0.9999);
                low += l[j]; high += h[j];
            }
            u64 cl_ = block_before64(low, low_all, sm.red), ch = block_before64(high, high_all, sm.red);
            const auto least = [&](u64 in_l, u64 in_h) { return fmax((double) in_l, (double) total - (double) (high_all - in_h)); };
            const auto most = [&](u64 in_l, u64 in_h) { return fmin((double) in_h, (double) total - (double) (low_all - in_l)); };
            u64 c = front;
            for (int j = 0; j < 4; j++) {
                if (most(cl_, ch) < want && most(cl_ + l[j], ch + h[j]) >= want) { sm.answer[0] = 4 * tid + j; sm.answer[2] = c; }
                if (least(cl_, ch) < want && least(cl_ + l[j], ch + h[j]) >= want) sm.answer[1] = 4 * tid + j;
                c += cnt[j]; cl_ += l[j]; ch += h[j];
            }
            __syncthreads();
            c = front;
            for (int j = 0; j < 4; j++) { c += cnt[j]; if (4 * tid + j == (int) sm.answer[1]) sm.answer[3] = c; }
        }
        __syncthreads();
        b_lo = (int) sm.answer[0]; b_hi = (int) sm.answer[1];
        int n_between = (int) (sm.answer[3] - sm.answer[2]);
        cl.sync();                                                       // bins have been read
        if (k > 0) {
            if (n_between <= SA_LIST) {
                gather([&](float v) { return bin_of(v) <= b_hi; });
                if (rank == 0) {
                    const int m = sorted(), per = (m + SA_THREADS - 1) / SA_THREADS, i0 = min(m, tid * per), i1 = min(m, i0 + per);
                    u64 mine_w = 0, all;
                    for (int i = i0; i < min(i1, k); i++) mine_w += weight(key_logit(list[i]));
                    u64 c = block_before64(mine_w, all, sm.red);
                    const double want = by_p ? (double) top_p * (double) all : 0.0;
                    for (int i = i0; i < min(i1, k); i++) {
                        // the last token that is kept: the sum in front of it is short of the share (the first always is kept)
                        const u64 w = weight(key_logit(list[i]));
                        const bool in = i == 0 || !by_p || (double) c < want, next = i + 1 < k && (!by_p || (double) (c + w) < want);
                        if (in && !next) sm.answer[0] = list[i];
                        c += w;
                    }
                    __syncthreads();
                    const u64 e = sm.answer[0];
                    if (tid < blocks) cl.map_shared_rank(&sm, tid)->edge = e;
                }
                cl.sync();
                edge = sm.edge;
            } else {
                edge = bisect(0, false, (double) k);
                if (by_p) { const double want = (double) top_p * (double) sum_from(edge); edge = want > 0.0 ? bisect(edge, true, want) : first; }
            }
        } else {
            const double want = (double) top_p * (double) total;
            u64 in_front = 0;                                            // sum of the bins in front of b_lo
            for (int i = tid; i < n; i += SA_THREADS) { const float v = logit(i); if (bin_of(v) < b_lo) in_front += weight(v); }
            in_front = cluster_join(cl, sm, in_front, 0ull, turn, add);
            float f_lo = (float) b_lo / SA_PER_NAT, f_scale = 0.f;
            int f_bin = -1;
            if (n_between > SA_LIST) {                                   // 2048 finer bins between b_lo and b_hi, their sums exact
                f_scale = SA_BINS * SA_PER_NAT / (float) (b_hi - b_lo + 1);
                int * count = reinterpret_cast<int *>(fine + SA_BINS);
                for (int i = tid; i < SA_BINS; i += SA_THREADS) { fine[i] = 0; count[i] = 0; }
                __syncthreads();
                for (int i = tid; i < n; i += SA_THREADS) {
                    const float v = logit(i);
                    const int b = bin_of(v);
                    if (b >= b_lo && b <= b_hi) {
                        const int fb = (int) fminf((below(v) - f_lo) * f_scale, (float) (SA_BINS - 1));
                        atomicAdd(&fine[fb], weight(v));
                        atomicAdd(&count[fb], 1);
                    }
                }
                cl.sync();
                u64 w[4] = {0, 0, 0, 0};
                int fc[4] = {0, 0, 0, 0};
                for (int r = 0; r < blocks; r++) {
                    const u64 * fw = cl.map_shared_rank(fine, r) + 4 * tid;
                    const int * ff = cl.map_shared_rank(count, r) + 4 * tid;
                    for (int j = 0; j < 4; j++) { w[j] += fw[j]; fc[j] += ff[j]; }
                }
                u64 c = in_front + block_before64(w[0] + w[1] + w[2] + w[3], dummy, sm.red);
                if (tid == 0) sm.answer[0] = SA_BINS;
                __syncthreads();
                for (int j = 0; j < 4; j++) {
                    if ((double) c < want && (double) (c + w[j]) >= want) { sm.answer[0] = 4 * tid + j; sm.answer[1] = c; sm.answer[2] = fc[j]; }
                    c += w[j];
                }
                __syncthreads();
                if (sm.answer[0] < SA_BINS) { f_bin = (int) sm.answer[0]; in_front = sm.answer[1]; n_between = (int) sm.answer[2]; }
                cl.sync();
            }
            if (n_between <= SA_LIST) {
                gather([&](float v) {
                    const int b = bin_of(v);
                    return b >= b_lo && b <= b_hi && (f_bin < 0 || (int) fminf((below(v) - f_lo) * f_scale, (float) (SA_BINS - 1)) == f_bin);
                });
                if (rank == 0) {
                    const int m = sorted(), per = (m + SA_THREADS - 1) / SA_THREADS, i0 = min(m, tid * per), i1 = min(m, i0 + per);
                    u64 mine_w = 0, all;
                    for (int i = i0; i < i1; i++) mine_w += weight(key_logit(list[i]));
                    u64 c = in_front + block_before64(mine_w, all, sm.red);
                    if (tid == 0) sm.answer[0] = m ? list[m - 1] : first;
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
            } else edge = want > 0.0 ? bisect(0, true, want) : first;
        }
    }
    // the draw: a warp sums its part of the slice, the parts stand in order of index
    const double cold = 1.0 / (double) temperature;
    const auto drawn = [&](int i) -> u64 {
        const float v = logit(i);
        if (below(v) > far || v == -INFINITY || order_key(v, base + i) < edge) return 0;
        const double x = exactly(v);
        if (min_p > 0.f && (double) fixed_weight(x) < (double) min_p * 1099511627776.0) return 0;
        return fixed_weight(x == 0.0 ? 0.0 : x * cold);
    };
    const int seg = (n + SA_WARPS - 1) / SA_WARPS, i0 = min(n, warp * seg), i1 = min(n, i0 + seg);
    u64 mine = 0;
    for (int i = i0 + lane; i < i1; i += 32) mine += drawn(i);
    mine = warp_reduce(mine, add);
    __syncthreads();
    if (lane == 0) sm.red[warp] = mine;
    __syncthreads();
    u64 front = 0, block_sum = 0;
    for (int w = 0; w < SA_WARPS; w++) { if (w < warp) front += sm.red[w]; block_sum += sm.red[w]; }
    if (tid < blocks) cl.map_shared_rank(&sm, tid)->each[rank] = block_sum;
    cl.sync();
    u64 total = 0;
    for (int r = 0; r < blocks; r++) { if (r < rank) front += sm.each[r]; total += sm.each[r]; }
    const double at = (double) a.u[row] * (double) total;
    const u64 target = at >= (double) total ? total - 1 : at > 0.0 ? (u64) at : 0;
    if (front <= target && target < front + mine) {                      // one warp of the cluster
        u64 c = front;
        for (int i = i0; i < i1; i += 32) {
            u64 w = i + lane < i1 ? drawn(i + lane) : 0, up = w;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) { const u64 x = __shfl_up_sync(0xffffffffu, up, d); if (lane >= d) up += x; }
            const unsigned hit = __ballot_sync(0xffffffffu, c + up > target);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    const double x = exactly(logit(i + lane));
                    finish(base + i + lane, (float) (-(x == 0.0 ? 0.0 : x * cold) - log((double) total * 0x1p-40)));
                }
                break;
            }
            c += __shfl_sync(0xffffffffu, up, 31);
        }
    }
    cl.sync();
}

}  // namespace srv
}  // namespace b200
