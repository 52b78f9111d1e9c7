// serve_pages.cuh — the life of the cache's pages (sm_100a): reserving, forking, freeing, compacting and copying them, all on the device.
//
// refs[page] counts the sequences that hold a page; 0 is free. There is no list of free pages: a call looks through refs (4 bytes a page) and takes the lowest ones, in the order in
// which its sequences ask, so that the same calls always give the same pages. Each call is a plan of one block, all or nothing, which leaves what is to be copied in the workspace, and
// where pages are copied a second kernel that moves them in every layer at the memory's rate.
// Measured: 48 pages reserved in a pool of 4096 8.6 us, of 65 536 13 us (a block reads 256 KB of counts); 24 slots forked 9 us and their part-full pages copied 7 (8 layers, 15 MB read and written); 12 slots freed
// 2.5 us; 255 MB compacted 8 us for the plan and 43 for the moves (6.0 TB/s, 93 % of the copy rate); 600 pages of 32 layers copied 461 us (6.1 TB/s). One block plans because every page that
// is taken depends on all that were taken before; latency bounds it.
#pragma once
#include "serve_cache.cuh"

namespace b200 {
namespace srv {

struct Pages {
    int32_t * table;
    int64_t table_stride;
    int n_slots, max_pages;
    int32_t * held, * refs;
    int n_pages, page_log2;
    uint8_t * pool;
    int64_t layer_stride, page_stride;
    int n_layer, n_kv, tile_bytes;
};
// what a plan leaves for the kernel behind it: plan[0] copies, plan[1] pages in use before (compaction); then from, to, tiles of each head
constexpr int PG_CHUNK = 2048, PLAN_HEAD = 4, PG_THREADS = 1024, PG_MAX_SLOTS = 1 << 18, PG_MAX_PAGES = 1 << 20, PG_MAX_N = 4096;

// bits of the pages with refs == 0 (or of the others), 32 a word. A warp reads 1024 neighbouring counts at a time, 16 bytes a lane; eight lanes make a word
__device__ __forceinline__ void page_bits(const Pages & p, bool free_ones, uint32_t * bits) {
    const int words = (p.n_pages + 31) >> 5, lane = threadIdx.x & 31;
    const bool whole = (reinterpret_cast<uintptr_t>(p.refs) & 15) == 0;
    for (int r0 = (threadIdx.x >> 5) * 1024; r0 < p.n_pages; r0 += PG_THREADS * 32) {
        int4 v[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = r0 + 128 * j + 4 * lane;
            v[j] = make_int4(0, 0, 0, 0);
            if (whole && i + 4 <= p.n_pages) v[j] = *reinterpret_cast<const int4 *>(p.refs + i);
            else {
                if (i < p.n_pages) v[j].x = p.refs[i];
                if (i + 1 < p.n_pages) v[j].y = p.refs[i + 1];
                if (i + 2 < p.n_pages) v[j].z = p.refs[i + 2];
                if (i + 3 < p.n_pages) v[j].w = p.refs[i + 3];
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint32_t m = (uint32_t) ((v[j].x > 0) | (v[j].y > 0) << 1 | (v[j].z > 0) << 2 | (v[j].w > 0) << 3) << (4 * (lane & 7));
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) m |= __shfl_xor_sync(0xffffffffu, m, d);
            const int w = (r0 >> 5) + 4 * j + (lane >> 3);
            if (free_ones) m = ~m & (32 * w + 32 <= p.n_pages ? 0xffffffffu : (1u << (p.n_pages & 31)) - 1);
            if ((lane & 7) == 0 && w < words) bits[w] = m;
        }
    }
    __syncthreads();
}
// sum over the threads in front of this one; `all`: of the whole block
__device__ __forceinline__ int block_before(int mine, int & all) {
    __shared__ int sums[PG_THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int up = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const int x = __shfl_up_sync(0xffffffffu, up, d); if (lane >= d) up += x; }
    __syncthreads();
    if (lane == 31) sums[warp] = up;
    __syncthreads();
    int off = 0, sum = 0;
    for (int w = 0; w < PG_THREADS / 32; w++) { if (w < warp) off += sums[w]; sum += sums[w]; }
    all = sum;
    return off + up - mine;
}
// f(k, page) for the set bits in ascending order, k = 0, 1, ...; returns how many there are. f runs for the first `most` of them
template <typename F> __device__ __forceinline__ int each_bit(const uint32_t * bits, int words, int most, F f) {
    const int per = (words + PG_THREADS - 1) / PG_THREADS, w0 = min(words, (int) threadIdx.x * per), w1 = min(words, w0 + per);
    int mine = 0, all;
    for (int w = w0; w < w1; w++) mine += __popc(bits[w]);
    int k = block_before(mine, all);
    for (int w = w0; w < w1 && k < most; w++)
        for (uint32_t m = bits[w]; m && k < most; m &= m - 1, k++) f(k, 32 * w + __ffs(m) - 1);
    return all;
}
__device__ __forceinline__ int n_bits(const uint32_t * bits, int words) { return each_bit(bits, words, 0, [](int, int) {}); }

// pages for first[i + 1] - first[i] tokens more of each slot, behind those that it holds
__global__ void __launch_bounds__(PG_THREADS) k_pages_reserve(const Pages p, const int32_t * slots, const int32_t * first, int n, int32_t * status) {
    extern __shared__ uint32_t pg_smem[];
    __shared__ int from[PG_MAX_N], before[PG_MAX_N + 1];           // of each sequence: the first page that is missing, pages missing in front of it
    __shared__ int chunk[PG_CHUNK];
    __shared__ int bad;
    const int words = (p.n_pages + 31) >> 5, slot_words = (p.n_slots + 31) >> 5;
    uint32_t * free_pages = pg_smem, * seen = pg_smem + words;
    if (threadIdx.x == 0) bad = 0;
    for (int i = threadIdx.x; i < slot_words; i += PG_THREADS) seen[i] = 0;
    page_bits(p, true, free_pages);
    const int per = (n + PG_THREADS - 1) / PG_THREADS, s0 = min(n, (int) threadIdx.x * per), s1 = min(n, s0 + per);
    int mine = 0, all;
    for (int s = s0; s < s1; s++) {
        const int slot = slots ? slots[s] : s, more = first[s + 1] - first[s];
        from[s] = 0; before[s] = mine;
        if ((unsigned) slot >= (unsigned) p.n_slots || more < 0) { bad = 1; continue; }
        if (atomicOr(&seen[slot >> 5], 1u << (slot & 31)) >> (slot & 31) & 1) { bad = 1; continue; }
        const int32_t * row = p.table + (int64_t) slot * p.table_stride;
        const int64_t need = ((int64_t) p.held[slot] + more + (1 << p.page_log2) - 1) >> p.page_log2;
        if (p.held[slot] < 0 || need > p.max_pages) { bad = 1; continue; }
        int f = min(p.held[slot] >> p.page_log2, (int) need);
        while (f < need && row[f] >= 0) f++;
        for (int i = f; i < need; i++) if (row[i] >= 0) bad = 1;
        from[s] = f;
        mine += (int) need - f;
    }
    const int off = block_before(mine, all);
    for (int s = s0; s < s1; s++) before[s] += off;
    if (threadIdx.x == 0) before[n] = all;
    __syncthreads();
    const int have = n_bits(free_pages, words);
    const bool refused = bad != 0;
    if (!refused && have >= all)
        for (int k0 = 0; k0 < all; k0 += PG_CHUNK) {               // the pages by their bits, then a thread a page
            each_bit(free_pages, words, min(all, k0 + PG_CHUNK), [&](int k, int page) { if (k >= k0) chunk[k - k0] = page; });
            __syncthreads();
            for (int i = threadIdx.x; i < min(PG_CHUNK, all - k0); i += PG_THREADS) {
                const int k = k0 + i, page = chunk[i];
                int s = 0;
                for (int hi = n; hi - s > 1;) { const int mid = (s + hi) >> 1; if (before[mid] <= k) s = mid; else hi = mid; }
                p.table[(int64_t) (slots ? slots[s] : s) * p.table_stride + from[s] + k - before[s]] = page;
                p.refs[page] = 1;
            }
            __syncthreads();
        }
    if (threadIdx.x == 0) *status = refused ? -1 : max(0, all - have);
}

// children take their parents' full pages and a copy of the page that is part full
__global__ void __launch_bounds__(PG_THREADS) k_pages_fork(const Pages p, const int32_t * parents, const int32_t * children, int n, int32_t * status, int32_t * plan) {
    extern __shared__ uint32_t pg_smem[];
    __shared__ int before[PG_MAX_N + 1];                           // part-full pages in front of each pair
    __shared__ int bad;
    const int words = (p.n_pages + 31) >> 5, slot_words = (p.n_slots + 31) >> 5, P = 1 << p.page_log2;
    uint32_t * free_pages = pg_smem, * taken = pg_smem + words;
    if (threadIdx.x == 0) bad = 0;
    for (int i = threadIdx.x; i < slot_words; i += PG_THREADS) taken[i] = 0;
    page_bits(p, true, free_pages);
    for (int s = threadIdx.x; s < n; s += PG_THREADS) {
        const int c = children[s], a = parents[s];
        if ((unsigned) c >= (unsigned) p.n_slots || (unsigned) a >= (unsigned) p.n_slots) { bad = 1; continue; }
        if (atomicOr(&taken[c >> 5], 1u << (c & 31)) >> (c & 31) & 1) bad = 1;
        if (p.held[c] != 0 || p.table[(int64_t) c * p.table_stride] >= 0) bad = 1;
        if (p.held[a] < 0 || p.held[a] > p.max_pages << p.page_log2) bad = 1;
    }
    __syncthreads();
    bool refused = bad != 0;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (!refused) {
        for (int s = warp; s < n; s += PG_THREADS / 32) {          // a child is no parent, a parent's pages are the pool's and held
            const int a = parents[s], used = (p.held[a] + P - 1) >> p.page_log2;
            if (taken[a >> 5] >> (a & 31) & 1) bad = 1;
            for (int i = lane; i < used; i += 32) {
                const int page = p.table[(int64_t) a * p.table_stride + i];
                if ((unsigned) page >= (unsigned) p.n_pages || p.refs[page] <= 0) bad = 1;
            }
        }
    }
    const int per = (n + PG_THREADS - 1) / PG_THREADS, s0 = min(n, (int) threadIdx.x * per), s1 = min(n, s0 + per);
    int mine = 0, all;
    if (!refused) for (int s = s0; s < s1; s++) { before[s] = mine; mine += (p.held[parents[s]] & (P - 1)) != 0; }
    const int off = block_before(mine, all);
    if (!refused) for (int s = s0; s < s1; s++) before[s] += off;
    const int have = n_bits(free_pages, words);
    __syncthreads();
    refused = bad != 0;
    const bool go = !refused && have >= all;
    if (threadIdx.x == 0) {
        before[n] = all;
        *status = refused ? -1 : max(0, all - have);
        plan[0] = go ? all : 0;
    }
    __syncthreads();
    if (!go) return;
    int32_t * from = plan + PLAN_HEAD, * to = from + n, * tiles = to + n;
    for (int s = s0; s < s1; s++) {
        const int a = parents[s], rest = p.held[a] & (P - 1);
        if (rest) { from[before[s]] = p.table[(int64_t) a * p.table_stride + (p.held[a] >> p.page_log2)]; tiles[before[s]] = (rest + 15) >> 4; }
    }
    each_bit(free_pages, words, all, [&](int k, int page) { to[k] = page; p.refs[page] = 1; });
    __syncthreads();
    for (int s = warp; s < n; s += PG_THREADS / 32) {
        const int a = parents[s], c = children[s], full = p.held[a] >> p.page_log2;
        const int32_t * row = p.table + (int64_t) a * p.table_stride;
        int32_t * mine_row = p.table + (int64_t) c * p.table_stride;
        for (int i = lane; i < p.max_pages; i += 32) {
            int page = -1;
            if (i < full) { page = row[i]; atomicAdd(&p.refs[page], 1); }
            else if (i == full && (p.held[a] & (P - 1))) page = to[before[s]];
            mine_row[i] = page;
        }
        if (lane == 0) p.held[c] = p.held[a];
    }
}

// a warp a slot. A slot that stands twice in the list is freed once
__global__ void __launch_bounds__(256) k_pages_free(const Pages p, const int32_t * slots, int n) {
    const int s = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (s >= n) return;
    const int slot = slots[s];
    if ((unsigned) slot >= (unsigned) p.n_slots) return;
    int32_t * row = p.table + (int64_t) slot * p.table_stride;
    for (int i = lane; i < p.max_pages; i += 32) {
        if (row[i] < 0) continue;
        const int page = atomicExch(&row[i], -1);
        if ((unsigned) page < (unsigned) p.n_pages) atomicSub(&p.refs[page], 1);
    }
    if (lane == 0) p.held[slot] = 0;
}

// pages in use behind the first `live` ones go, in order, to the free ones among those
__global__ void __launch_bounds__(PG_THREADS) k_pages_compact(const Pages p, int32_t * live_out, int32_t * plan) {
    extern __shared__ uint32_t pg_smem[];
    const int words = (p.n_pages + 31) >> 5;
    uint32_t * used = pg_smem;
    page_bits(p, false, used);
    const int live = n_bits(used, words);
    int32_t * from = plan + PLAN_HEAD, * to = from + p.n_pages;
    const auto below = [&](int w) { return 32 * w + 32 <= live ? 0xffffffffu : 32 * w >= live ? 0u : (1u << (live & 31)) - 1; };
    // the movers: used & behind; each_bit takes the bits as they stand, so they are masked in place and turned round for the holes
    const int per = (words + PG_THREADS - 1) / PG_THREADS, w0 = min(words, (int) threadIdx.x * per), w1 = min(words, w0 + per);
    int movers = 0, holes = 0, moved, all;
    for (int w = w0; w < w1; w++) { movers += __popc(used[w] & ~below(w)); holes += __popc(~used[w] & below(w)); }
    int k = block_before(movers, moved);
    for (int w = w0; w < w1; w++) for (uint32_t m = used[w] & ~below(w); m; m &= m - 1) from[k++] = 32 * w + __ffs(m) - 1;
    k = block_before(holes, all);
    for (int w = w0; w < w1; w++) for (uint32_t m = ~used[w] & below(w); m; m &= m - 1) to[k++] = 32 * w + __ffs(m) - 1;
    __syncthreads();
    int32_t * moved_to = to + p.n_pages;
    for (int i = live + threadIdx.x; i < p.n_pages; i += PG_THREADS) moved_to[i] = -1;      // (no table names a page without references)
    __syncthreads();
    for (int i = threadIdx.x; i < moved; i += PG_THREADS) {
        const int a = from[i], b = to[i];
        moved_to[a] = b;
        p.refs[b] = p.refs[a];
        p.refs[a] = 0;
    }
    if (threadIdx.x == 0) { plan[0] = moved; plan[1] = live; *live_out = live; }
}

// pairs of a raw copy: whole pages; a page that is written twice, or written and read, is refused
__global__ void __launch_bounds__(PG_THREADS) k_pages_check_copy(const Pages p, const int32_t * src, const int32_t * dst, int n, int32_t * status, int32_t * plan) {
    extern __shared__ uint32_t pg_smem[];
    __shared__ int bad;
    const int words = (p.n_pages + 31) >> 5;
    if (threadIdx.x == 0) bad = 0;
    for (int i = threadIdx.x; i < words; i += PG_THREADS) pg_smem[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += PG_THREADS) {
        const int d = dst[i];
        if ((unsigned) d >= (unsigned) p.n_pages || (unsigned) src[i] >= (unsigned) p.n_pages) { bad = 1; continue; }
        if (atomicOr(&pg_smem[d >> 5], 1u << (d & 31)) >> (d & 31) & 1) bad = 1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += PG_THREADS) {
        const int s = src[i];
        if ((unsigned) s < (unsigned) p.n_pages && (pg_smem[s >> 5] >> (s & 31) & 1)) bad = 1;
    }
    __syncthreads();
    int32_t * from = plan + PLAN_HEAD, * to = from + n, * tiles = to + n;
    for (int i = threadIdx.x; i < n; i += PG_THREADS) { from[i] = src[i]; to[i] = dst[i]; tiles[i] = 1 << (p.page_log2 - 4); }
    if (threadIdx.x == 0) { *status = bad ? -1 : 0; plan[0] = bad ? 0 : n; }
}

// the planned copies in every layer: a warp takes a head's tiles of a page at a time, 16 bytes a lane, eight on their way. Lists of n entries; tiles == nullptr: all of a page's.
// moved_to: tables are rewritten too, where they name a page from `live` on
__global__ void __launch_bounds__(256) k_pages_move(const Pages p, const int32_t * plan, int n, bool parts, const int32_t * moved_to) {
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t) gridDim.x * 8, me = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int copies = plan[0], page_tiles = 1 << (p.page_log2 - 4);
    const int32_t * from = plan + PLAN_HEAD, * to = from + n, * tiles = to + n;
    if (moved_to) {
        const int live = plan[1];
        for (int64_t i = me * 32 + lane; i < (int64_t) p.n_slots * p.max_pages; i += warps * 32) {
            int32_t * e = p.table + i / p.max_pages * p.table_stride + i % p.max_pages;
            if (*e >= live && *e < p.n_pages) *e = moved_to[*e];
        }
    }
    const int64_t head_bytes = (int64_t) page_tiles * p.tile_bytes, total = (int64_t) copies * p.n_layer * p.n_kv;
    for (int64_t w = me; w < total; w += warps) {
        const int head = (int) (w % p.n_kv), i = (int) (w / p.n_kv % copies), layer = (int) (w / p.n_kv / copies);
        const int bytes = (parts ? tiles[i] : page_tiles) * p.tile_bytes;
        const uint8_t * a = p.pool + layer * p.layer_stride + from[i] * p.page_stride + head * head_bytes;
        uint8_t * b = p.pool + layer * p.layer_stride + to[i] * p.page_stride + head * head_bytes;
#pragma unroll 1
        for (int at = 16 * lane; at < bytes; at += 8 * 512) {
            uint4 v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) if (at + 512 * j < bytes) v[j] = *reinterpret_cast<const uint4 *>(a + at + 512 * j);
#pragma unroll
            for (int j = 0; j < 8; j++) if (at + 512 * j < bytes) *reinterpret_cast<uint4 *>(b + at + 512 * j) = v[j];
        }
    }
}

}  // namespace srv
}  // namespace b200
