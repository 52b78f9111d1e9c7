// serve_pages.cuh — the life of the cache's pages (sm_100a): reserving, forking, freeing, compacting and copying them, all on the device.
//
// refs[page] counts the sequences that hold a page; 0 is free. There is no list of free pages: a call looks through refs (4 bytes a page) and takes the lowest ones, in the order in
// which its sequences ask, so that the same calls always give the same pages. Each call is a plan of one block, all or nothing, which leaves what is to be copied in the workspace, and
// where pages are copied a second kernel that moves them in every layer at the memory's rate.
// Measured: 48 pages reserved in a pool of 4096 8.6 us, of 65 536 13 us (a block reads 256 KB of counts); 24 slots forked 9 us and their part-full pages copied 7 (8 layers, 15 MB read and written); 12 slots freed
// 2.5 us; 255 MB compacted 8 us for the plan and 43 for the moves (6.0 TB/s, 93 % of the copy rate); 600 pages of 32 layers copied 461 us (6.1 TB/s). One block plans because every page that
// is taken depends on all that were taken before; latency bounds it. Tables of a step: 48 sequences in 4096 pages 9.6 us for the plan and 2.4 for what is trimmed, 300 (three with 900 rows) in 60 000
// pages 12.3 and 2.5.
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
template <typename V> __device__ __forceinline__ V block_before(V mine, V & all) {
    __shared__ V sums[PG_THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V up = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const V x = __shfl_up_sync(0xffffffffu, up, d); if (lane >= d) up += x; }
    __syncthreads();
    if (lane == 31) sums[warp] = up;
    __syncthreads();
    V off = 0, sum = 0;
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

// The tables of a step from its rows' numbers: first, the pages that k_pages_reserve would take, and of each row its position and its place (page x page_tokens + token) in a layer's pool.
// One block, since every page that is taken depends on all that were taken before; latency bounds it, so loads that do not depend on one another are asked for together: the first 32 768 counts of
// pages (more are looked at only where those do not have enough free ones) with the sequences' own numbers, of a sequence's row of the table four entries by its thread and, of long portions, the
// others by a warp. Up to PLAN_ROWS rows are the block's own to write, more are another kernel's.
constexpr int PLAN_ROWS = 4096, PLAN_PAGES = PG_THREADS * 32, PLAN_OWN = 4;
__host__ __device__ constexpr size_t plan_bytes(int n) { return 4 * ((size_t) 6 * n + 2 + PG_CHUNK); }
// sums over the threads in front of this one, and of the block
__device__ __forceinline__ void block_before2(long long x, long long y, long long & x_front, long long & x_all, long long & y_front, long long & y_all) {
    __shared__ long long sums[2][PG_THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long up = x, vp = y;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, up, d), v = __shfl_up_sync(0xffffffffu, vp, d);
        if (lane >= d) { up += u; vp += v; }
    }
    __syncthreads();
    if (lane == 31) { sums[0][warp] = up; sums[1][warp] = vp; }
    __syncthreads();
    long long u = sums[0][lane], v = sums[1][lane], u0 = u, v0 = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long w = __shfl_up_sync(0xffffffffu, u, d), z = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) { u += w; v += z; }
    }
    x_all = __shfl_sync(0xffffffffu, u, 31); y_all = __shfl_sync(0xffffffffu, v, 31);
    x_front = up - x + __shfl_sync(0xffffffffu, u - u0, warp);
    y_front = vp - y + __shfl_sync(0xffffffffu, v - v0, warp);
}
// the counts of pages p0 + 1024 warp + .., 32 a lane, and the word of free ones among page p0 + 1024 warp + 32 lane + 0 .. 31
__device__ __forceinline__ void counts_begun(const Pages & p, int p0, bool whole, int4 (&v)[8]) {
    const int lane = threadIdx.x & 31, r0 = p0 + (int) (threadIdx.x >> 5) * 1024;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = r0 + 128 * j + 4 * lane;
        v[j] = make_int4(1, 1, 1, 1);
        if (whole && i + 4 <= p.n_pages) v[j] = *reinterpret_cast<const int4 *>(p.refs + i);
        else {
            if (i < p.n_pages) v[j].x = p.refs[i];
            if (i + 1 < p.n_pages) v[j].y = p.refs[i + 1];
            if (i + 2 < p.n_pages) v[j].z = p.refs[i + 2];
            if (i + 3 < p.n_pages) v[j].w = p.refs[i + 3];
        }
    }
}
__device__ __forceinline__ uint32_t counts_word(const int4 (&v)[8]) {
    const int lane = threadIdx.x & 31;
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        uint32_t m = (uint32_t) ((v[j].x <= 0) | (v[j].y <= 0) << 1 | (v[j].z <= 0) << 2 | (v[j].w <= 0) << 3) << (4 * (lane & 7));
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) m |= __shfl_xor_sync(0xffffffffu, m, d);
        const uint32_t got = __shfl_sync(0xffffffffu, m, (lane & 3) * 8);          // word 4 j + lane % 4
        if (lane >> 2 == j) mine = got;
    }
    return mine;
}
struct PlanSeqs { const int32_t * first, * slot, * held; };          // of the step's sequences; slot -1: none that can be
__device__ __forceinline__ void row_place(const Pages & p, const PlanSeqs & q, int n, int r, int & pos, int & place) {
    pos = place = -1;
    if (n <= 0 || r >= q.first[n]) return;
    int s = 0;                                                       // the last sequence that begins at or before r
    for (int hi = n; hi - s > 1;) { const int mid = (s + hi) >> 1; if (q.first[mid] <= r) s = mid; else hi = mid; }
    const int slot = q.slot[s], held = q.held[s];
    if (slot < 0 || held < 0) return;
    const long long at = (long long) held + r - q.first[s], i = at >> p.page_log2;
    pos = (int) min(at, (long long) INT32_MAX);
    const int page = i < p.max_pages ? p.table[(int64_t) slot * p.table_stride + i] : -1;
    if ((unsigned) page < (unsigned) p.n_pages) place = (page << p.page_log2) + (pos & ((1 << p.page_log2) - 1));
}
static __global__ void __launch_bounds__(PG_THREADS) k_pages_plan(const Pages p, const int32_t * slots, const int32_t * counts, int n, int n_rows, int32_t * first_out, int32_t * positions,
                                                                  int32_t * places, int32_t * status, bool rows_too) {
    extern __shared__ uint32_t pg_smem[];
    __shared__ int bad, n_long;
    const int slot_words = (p.n_slots + 31) >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t * seen = pg_smem;
    int32_t * first = reinterpret_cast<int32_t *>(seen + slot_words), * from = first + n + 1, * before = from + n, * slot_of = before + n + 1, * held_of = slot_of + n, * long_of = held_of + n,
            * chunk = long_of + n;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const bool whole = (reinterpret_cast<uintptr_t>(p.refs) & 15) == 0;
    int4 v[8];
    counts_begun(p, 0, whole, v);
    const int per = (n + PG_THREADS - 1) / PG_THREADS, s0 = min(n, (int) threadIdx.x * per), s1 = min(n, s0 + per);
    for (int i = threadIdx.x; i < slot_words; i += PG_THREADS) seen[i] = 0;
    if (threadIdx.x == 0) { bad = 0; n_long = 0; }
    __syncthreads();
    // of each sequence: pages that its rows need and, of those, the first that is missing
    const auto needs = [&](int held, int more) { return ((int64_t) held + more + (1 << p.page_log2) - 1) >> p.page_log2; };
    for (int s = s0; s < s1; s++) {
        int slot = slots ? slots[s] : s;
        const int more = counts[s];
        if ((unsigned) slot >= (unsigned) p.n_slots) slot = -1;
        const int held = slot >= 0 ? p.held[slot] : -1;
        slot_of[s] = slot; held_of[s] = held; from[s] = 0;
        if (slot < 0 || more < 0 || held < 0 || needs(held, more) > p.max_pages) { bad = 1; continue; }
        if (atomicOr(&seen[slot >> 5], 1u << (slot & 31)) >> (slot & 31) & 1) bad = 1;
        const int need = (int) needs(held, more), f = min(held >> p.page_log2, need);
        const int32_t * row = p.table + (int64_t) slot * p.table_stride;
        int e[PLAN_OWN], at = f;
#pragma unroll
        for (int i = 0; i < PLAN_OWN; i++) e[i] = f + i < need ? row[f + i] : -1;
#pragma unroll
        for (int i = 0; i < PLAN_OWN; i++) {
            if (e[i] >= 0 && at < f + i) bad = 1;                    // a page behind one that is missing
            if (e[i] >= 0) at = f + i + 1;
        }
        from[s] = at;
        if (need - f > PLAN_OWN) long_of[atomicAdd(&n_long, 1)] = s;
    }
    const uint32_t free_word = counts_word(v);
    __syncthreads();
    for (int k = warp; k < n_long; k += PG_THREADS / 32) {           // the entries of long portions behind their first ones
        const int s = long_of[k], held = held_of[s], need = (int) needs(held, counts[s]), f = (held >> p.page_log2) + PLAN_OWN;
        const int32_t * row = p.table + (int64_t) slot_of[s] * p.table_stride;
        int at = from[s];
        bool hole = at < f;
        for (int i0 = f; i0 < need; i0 += 128) {
            int e[4];
#pragma unroll
            for (int j = 0; j < 4; j++) { const int i = i0 + 32 * j + lane; e[j] = i < need ? row[i] : -1; }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned there = __ballot_sync(0xffffffffu, e[j] >= 0);
                const int run = there == 0xffffffffu ? 32 : __ffs(~there) - 1;        // pages in front of the first that is missing
                if (there && (hole || (run < 32 && there >> run))) { if (lane == 0) bad = 1; }
                if (!hole) { at += run; hole = run < 32; }
            }
        }
        if (lane == 0) from[s] = min(at, need);
    }
    __syncthreads();
    long long mine = 0, rows = 0, front, all, row_front, all_rows;
    for (int s = s0; s < s1; s++) {
        const int more = counts[s];
        rows += min(max(more, 0), n_rows + 1);
        if (slot_of[s] >= 0 && more >= 0 && held_of[s] >= 0 && needs(held_of[s], more) <= p.max_pages) mine += needs(held_of[s], more) - from[s];
    }
    block_before2(mine, rows, front, all, row_front, all_rows);
    for (int s = s0; s < s1; s++) {
        const int more = counts[s];
        before[s] = (int) min(front, (long long) INT32_MAX);
        first[s] = (int) min(row_front, (long long) n_rows);
        row_front += min(max(more, 0), n_rows + 1);
        if (slot_of[s] >= 0 && more >= 0 && held_of[s] >= 0 && needs(held_of[s], more) <= p.max_pages) front += needs(held_of[s], more) - from[s];
    }
    if (threadIdx.x == 0) { before[n] = (int) min(all, (long long) INT32_MAX); first[n] = (int) min(all_rows, (long long) n_rows); if (all_rows > n_rows) bad = 1; }
    __syncthreads();
    for (int s = threadIdx.x; s <= n; s += PG_THREADS) first_out[s] = first[s];
    const bool refused = bad != 0;
    // whether there are as many free pages, looked for as far as need be
    long long have = 0, dummy, got, dummy_all;
    int looked = 0;
    uint32_t word = free_word;
    for (int p0 = 0; p0 < p.n_pages && have < all; p0 += PLAN_PAGES) {
        if (p0) { counts_begun(p, p0, whole, v); word = counts_word(v); }
        block_before2(__popc(word), 0, front, got, dummy, dummy_all);
        have += got;
        looked++;
    }
    if (!refused && have >= all && all > 0) {
        long long k0 = 0;                                            // free pages in front of the chunk
        for (int p0 = 0; k0 < all; p0 += PLAN_PAGES) {
            if (looked > 1) {
                counts_begun(p, p0, whole, v);
                word = counts_word(v);
                block_before2(__popc(word), 0, front, got, dummy, dummy_all);
            }
            // (the counts of this chunk are read; those that change are behind the barriers of the next)
            for (int c0 = 0; c0 < got && k0 + c0 < all; c0 += PG_CHUNK) {             // the pages by their bits, then a thread a page
                int k = (int) front;
                for (uint32_t m = word; m && k < c0 + PG_CHUNK; m &= m - 1, k++) if (k >= c0) chunk[k - c0] = p0 + 32 * (int) threadIdx.x + __ffs(m) - 1;
                __syncthreads();
                for (int i = threadIdx.x; i < min((long long) PG_CHUNK, min(got - c0, all - k0 - c0)); i += PG_THREADS) {
                    const int k = (int) (k0 + c0 + i), page = chunk[i];
                    int s = 0;
                    for (int hi = n; hi - s > 1;) { const int mid = (s + hi) >> 1; if (before[mid] <= k) s = mid; else hi = mid; }
                    p.table[(int64_t) slot_of[s] * p.table_stride + from[s] + k - before[s]] = page;
                    p.refs[page] = 1;
                }
                __syncthreads();
            }
            k0 += got;
        }
    }
    if (threadIdx.x == 0) *status = refused ? -1 : (int) min(max(0ll, all - have), (long long) INT32_MAX);
    if (rows_too) {
        constexpr int U = PLAN_ROWS / PG_THREADS;
        int pos[U], place[U];
#pragma unroll
        for (int u = 0; u < U; u++) { const int r = threadIdx.x + u * PG_THREADS; if (r < n_rows) row_place(p, PlanSeqs{first, slot_of, held_of}, n, r, pos[u], place[u]); }
#pragma unroll
        for (int u = 0; u < U; u++) { const int r = threadIdx.x + u * PG_THREADS; if (r < n_rows) { positions[r] = pos[u]; places[r] = place[u]; } }
    }
}
static __global__ void __launch_bounds__(256) k_pages_places(const Pages p, const int32_t * slots, const int32_t * first, int n, int n_rows, int32_t * positions, int32_t * places) {
    extern __shared__ uint32_t pg_smem[];
    int32_t * first_s = reinterpret_cast<int32_t *>(pg_smem), * slot_of = first_s + n + 1, * held_of = slot_of + n;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int s = threadIdx.x; s <= n; s += 256) {
        first_s[s] = first[s];
        if (s == n) break;
        const int slot = slots ? slots[s] : s;
        const bool in = (unsigned) slot < (unsigned) p.n_slots;
        slot_of[s] = in ? slot : -1;
        held_of[s] = in ? p.held[slot] : -1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = blockIdx.x * 1024 + i * 256 + threadIdx.x;
        int pos, place;
        if (r < n_rows) { row_place(p, PlanSeqs{first_s, slot_of, held_of}, n, r, pos, place); positions[r] = pos; places[r] = place; }
    }
}

// Pages that no row to come sees go back: those behind the tokens that are held (rows that were refused), and under a window those that lie whole in front of what the next row sees and behind
// the first `sinks` tokens. A warp 256 entries of a slot, all asked for together; a slot that stands twice in the list is looked at twice, its pages go once
static __global__ void __launch_bounds__(256) k_pages_trim(const Pages p, const int32_t * slots, int n, int window, int sinks) {
    const int64_t item = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31, parts = (p.max_pages + 255) >> 8, s = (int) (item / parts), i0 = (int) (item % parts) * 256 + lane;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (s >= n) return;
    const int slot = slots[s];
    if ((unsigned) slot >= (unsigned) p.n_slots) return;
    int32_t * row = p.table + (int64_t) slot * p.table_stride;
    int page[8];
#pragma unroll
    for (int j = 0; j < 8; j++) { const int i = i0 + 32 * j; page[j] = i < p.max_pages ? row[i] : -1; }
    const int P = 1 << p.page_log2, held = max(0, p.held[slot]), seen_from = window > 0 ? held - window + 1 : 0;
    const int full = (int) (((long long) held + P - 1) >> p.page_log2);                           // pages from this one on hold nothing
    const int hidden_from = window > 0 ? (int) (((long long) sinks + P - 1) >> p.page_log2) : 0, hidden_to = seen_from > 0 ? seen_from >> p.page_log2 : 0;      // pages of neither
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = i0 + 32 * j;
        if (page[j] >= 0 && (i >= full || (i >= hidden_from && i < hidden_to))) page[j] = atomicExch(&row[i], -1);
        else page[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) if ((unsigned) page[j] < (unsigned) p.n_pages) atomicSub(&p.refs[page[j]], 1);
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
        for (int s = warp; s < n; s += PG_THREADS / 32) {          // a child is no parent, a parent's pages are the pool's and held, or absent
            const int a = parents[s], used = (p.held[a] + P - 1) >> p.page_log2;
            if (taken[a >> 5] >> (a & 31) & 1) bad = 1;
            for (int i = lane; i < used; i += 32) {
                const int page = p.table[(int64_t) a * p.table_stride + i];
                if (page < 0 && i < p.held[a] >> p.page_log2) continue;      // a full page that k_pages_trim gave back: the child goes without it too
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
            if (i < full) { page = row[i]; if (page >= 0) atomicAdd(&p.refs[page], 1); }
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
