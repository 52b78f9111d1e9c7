// serve_attn.cuh — attention of a step's rows over the 4-bit cache (sm_100a): few rows of many sequences.
//
// A unit of work is a sequence's columns (a column is a row and a query head of one KV head: 8 NT of them) over the tiles of 16 tokens that its rows see. All units' tiles stand in one
// line, which is cut evenly over all warps of the grid: a warp walks its piece by itself, with the running maximum and sum of the soft-max in registers, and ends a unit that others share
// with a partial result that k_kv4_join adds. So sequences of any lengths fill the card, and nothing is waited for inside.
//   S^T = K Q^T: a tile's codes are the A operand of mma.sync (16 tokens x 16 dims), the columns the B operand. A block's 32 products are summed as codes and scaled once.
//   O^T += V^T P^T: V's codes times their scales (exact in fp16) are the A operand (16 dims x 16 tokens); P^T comes from S^T by movmatrix.
// Measured with 32 query heads on 8 of 128: HBM bounds long contexts (24 sequences of 12 000 to 32 000 tokens add 85 to 89 % of the copy rate's time), 10 to 13 us are the way to the first tile
// (launch, row, slot, page, codes) and the last parts: 48 sequences of 90 to 4090 tokens (116 MB) 35 us, 200 of 500 (115 MB) 40 us, 3 of 21 000 to 32 700 under 64 heads on 8 (99 MB) 31 us, one of 333 tokens 9.6 us with the join.
// Roundings: P to fp16 (2^-11, see P_LIFT); sums of scores and values, fp32 as the tensor cores add; the result. q is scaled by a power of two into fp16's range, which keeps its bits. With one
// column tile the codes' offset is taken off inside the sums of scores (FOLD): their terms are up to 1039 times q's entries, up to 8 times with two tiles and in serve_prompt.cuh. Seen where
// scores are very large: fp16 results for scores up to 169 are off by 1.80e-4 (rms; 1.65e-4 without, of which 1.59e-4 the result's rounding), up to 21 by 1.42e-4 either way. Without: 48 ragged
// sequences 35.1 us for 34.9, 3 long 31.2 for 30.7.
#pragma once
#include "serve_cache.cuh"

namespace b200 {
namespace srv {

template <typename T> struct alignas(16) Eight { T v[8]; };           // of 16-bit types
struct AttendArgs {
    Cache c;
    const void * q;
    int64_t q_row, q_head;
    bool q_whole;                        // eight entries of q stand on 16 bytes
    void * out;                          // [n_rows][n_head][HD]
    int group;
    float scale_log2;                    // scale x log2(e)
    int window;                          // 0: all positions
    int sinks;                           // first tokens that stay visible under a window (serve_kv16.cuh; the 4-bit cache has none)
    // workspace
    long long * before;                  // [n_seq + 1] pairs of tiles in front of each sequence; [n_seq + 1]: pairs of a warp's piece
    float * part, * ml;                  // [2 x warps][8 NT][HD], [2 x warps][8 NT][2]
};

constexpr int AT_WARPS = 4, AT_MAX_SEQ = 4096, AT_STAGES = 3, AT_OVER = 3;      // AT_OVER: what beginning a unit costs, in pairs of tiles (48 ragged sequences 49, 42, 38, 37, 37 us with 0 to 4)
__host__ __device__ constexpr int at_blocks(int nt) { return nt == 1 ? 3 : 2; }          // resident on an SM: 168 and 255 registers a thread
__host__ __device__ constexpr size_t at_ring_bytes(int hd) { return (size_t) AT_WARPS * AT_STAGES * 36 * hd; }
// P = 2^(score - base) is rounded to fp16, whose steps below 2^-14 are 2^-24. base is P_LIFT below the largest score, so that weights keep their 11 bits down to 2^-21 of the largest one, and what
// is left out of any is below 2^-32 of it: over 2^17 tokens behind one that takes most of the weight 2^-15 of the largest value, less than the output's rounding. base moves when a score passes the
// largest so far by 2^P_PASS; P stays within 2^15 until then. (2^4 and 11: 2^-36, but 48 ragged sequences 35.2 us for 34.9, 512 rows at 6000 74.0 for 70.5, 8192 rows 582 for 557)
constexpr float P_PASS = 8.f, P_LIFT = 7.f;
__device__ __forceinline__ uint32_t smem_at(const void * p) { return (uint32_t) __cvta_generic_to_shared(p); }
// 16 bytes from src, or zeros where bytes is 0
template <int AT> __device__ __forceinline__ void copy16(uint32_t dst, const uint8_t * src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0 + %3], [%1 + %3], 16, %2;" :: "r"(dst), "l"(src), "r"(bytes), "n"(AT) : "memory");
}
// where a lane copies a pair of tiles from: a for what lies in the first one, b in the second (less the first one's length), mid for the 512 bytes that hold the border
struct PairSrc { const uint8_t * a, * mid, * b; int bytes_a, bytes_mid, bytes_b; };
template <int HD> __device__ __forceinline__ void copy_pair(uint32_t dst, const PairSrc & s, int lane) {
    if constexpr (HD == 128) {
        copy16<0>(dst, s.a, s.bytes_a); copy16<512>(dst, s.a, s.bytes_a); copy16<1024>(dst, s.a, s.bytes_a); copy16<1536>(dst, s.a, s.bytes_a);
        copy16<2048>(dst, s.mid, s.bytes_mid);
        copy16<2560>(dst, s.b, s.bytes_b); copy16<3584>(dst, s.b, s.bytes_b); copy16<4096>(dst, s.b, s.bytes_b); copy16<2048 + 1024>(dst, s.b, s.bytes_b);
    } else {
        copy16<0>(dst, s.a, s.bytes_a); copy16<512>(dst, s.a, s.bytes_a);
        copy16<1024>(dst, s.mid, s.bytes_mid);
        copy16<1536>(dst, s.b, s.bytes_b);
        if (lane < 16) copy16<2048>(dst, s.b, s.bytes_b);
    }
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[2]) {       // d = a b + c, c of the two columns
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) { uint32_t r; asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x)); return r; }
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2 *>(&x); }
__device__ __forceinline__ uint32_t as_u(__half2 x) { return *reinterpret_cast<uint32_t *>(&x); }
__device__ __forceinline__ float exp2_fast(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// the eight codes of a word as pairs (n, n + 4) of nibbles over the last bits of 1024: 1024 + c for pairs 0 and 2, 1024 + 16 c for 1 and 3
__device__ __forceinline__ uint32_t pick(uint32_t w, uint32_t mask, uint32_t over) { uint32_t r; asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(over)); return r; }
__device__ __forceinline__ void codes8_raw(uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t x = i ? w >> 8 : w;
        p[2 * i] = pick(x, 0x000f000fu, 0x64006400u);
        p[2 * i + 1] = pick(x, 0x00f000f0u, 0x64006400u);
    }
}
// what a column's query is multiplied with: a power of two that brings its largest entry to 2^13 .. 2^14 (2^126 at most, of zeros too). An infinity's scores are infinities or NaN, whose
// soft-max is no number: they all become NaN, since negative ones look like masked ones
__device__ __forceinline__ float query_scale(float top) {
    const int e = (int) (__float_as_uint(top) >> 23);
    return e == 255 ? NAN : __uint_as_float((uint32_t) min(253, max(1, 267 - e)) << 23);
}
// less 8
__device__ __forceinline__ void codes8(uint32_t w, uint32_t (&p)[4]) {
    const __half2 eight = as_h2(0xe408e408u), sixteenth = as_h2(0x2c002c00u), seventy_two = as_h2(0xd480d480u);   // -1032, 1 / 16, -72
    codes8_raw(w, p);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        p[i] = as_u(__hadd2(as_h2(p[i]), eight));
        p[i + 1] = as_u(__hfma2(as_h2(p[i + 1]), sixteenth, seventy_two));
    }
}

// pairs of tiles [lo, lo + n) that the rows a .. b of a sequence see, one at least (it may have nothing to see in it)
struct Span { int lo, n; };
__device__ __forceinline__ Span span_of(const Cache & c, const Seq & q, int window, int a, int b) {
    const int last = min(q.held + b, (c.max_pages << c.page_log2) - 1);
    const int first = window > 0 ? max(0, q.held + a - window + 1) : 0;
    Span s;
    s.lo = first >> 5;
    s.n = q.slot < 0 || last < first ? 1 : (last >> 5) - s.lo + 1;
    return s;
}
// a sequence's units: column tiles x KV heads, of which each column tile has a span of its own. Units of a sequence are made equally long: the span of all its rows
__device__ __forceinline__ int col_tiles(const Seq & q, int group, int cols) { return (q.count * group + cols - 1) / cols; }

// (most quotients are of 31 bits)
__device__ __forceinline__ long long quotient(long long a, int b) { return a >> 31 ? a / b : (long long) ((unsigned) a / (unsigned) b); }

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(AT_WARPS * 32, at_blocks(NT)) k_kv4_attend(const AttendArgs a) {
    constexpr int NB = HD / 32, COLS = 8 * NT, TILE = 18 * HD, PAIR = 2 * TILE;
    constexpr bool FOLD = NT == 1;                                 // the codes' offsets are taken off in the sums, where there are registers for them
    extern __shared__ __align__(16) uint8_t at_raw[];              // each warp's ring of tiles, then before
    long long * before = reinterpret_cast<long long *>(at_raw + at_ring_bytes(HD));     // [n_seq + 1]
    __shared__ long long sums[AT_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3;
    const Cache & c = a.c;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // pairs of tiles in front of each sequence
    {
        constexpr int THREADS = AT_WARPS * 32, BATCH = 4;
        for (int b0 = tid; b0 < c.n_seq; b0 += THREADS * BATCH) {              // (slot, held, first: dependent reads, of four sequences at a time)
            Seq q[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; i++) q[i] = seq_at(c, min(b0 + i * THREADS, c.n_seq - 1));
#pragma unroll
            for (int i = 0; i < BATCH; i++)
                if (b0 + i * THREADS < c.n_seq)
                    before[b0 + i * THREADS] = q[i].count ? (long long) col_tiles(q[i], a.group, COLS) * c.n_kv * (span_of(c, q[i], a.window, 0, q[i].count - 1).n + AT_OVER) : 0;
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
        if (tid == AT_WARPS * 32 - 1) before[c.n_seq] = off + mine;
        __syncthreads();
    }
    const long long total = before[c.n_seq];
    const int n_warps = (int) gridDim.x * AT_WARPS;
    const long long per = max(1ll, quotient(total + n_warps - 1, n_warps));
    if (blockIdx.x == 0) {
        for (int s = tid; s <= c.n_seq; s += AT_WARPS * 32) a.before[s] = before[s];
        if (tid == 0) a.before[c.n_seq + 1] = per;
    }
    const int me = warp * (int) gridDim.x + (int) blockIdx.x;      // neighbouring pieces on different SMs
    long long at = me * per;
    const long long end = min(total, at + per);
    while (at < end) {
        int s = 0;
        for (int hi = c.n_seq; hi - s > 1;) { const int mid = (s + hi) >> 1; if (before[mid] <= at) s = mid; else hi = mid; }
        const Seq q = seq_at(c, s);
        const Span sp = span_of(c, q, a.window, 0, q.count - 1);               // (in pairs of tiles, like all counts here)
        const long long x = at - before[s];
        const int len = sp.n + AT_OVER, unit = (int) quotient(x, len), from = (int) (x - (long long) unit * len), to = (int) min((long long) len, from + (end - at));
        const int ct = unit / c.n_kv, head = unit - ct * c.n_kv, t0 = max(0, from - AT_OVER), t1 = to - AT_OVER;
        at += to - from;
        if (t1 <= 0) continue;
        // the columns' queries: asked for ahead of the pages
        Eight<T> raw[NT][NB] = {};
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int col = ct * COLS + 8 * n + g, i = col / a.group, h = head * a.group + col - i * a.group;
            if (i >= q.count) continue;
            const T * qp = static_cast<const T *>(a.q) + (q.begin + i) * a.q_row + h * a.q_head + 8 * tq;
            if (a.q_whole) {
#pragma unroll
                for (int b = 0; b < NB; b++) raw[n][b] = *reinterpret_cast<const Eight<T> *>(qp + 32 * b);
            } else {
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int j = 0; j < 8; j++) raw[n][b].v[j] = qp[32 * b + j];
            }
        }
        // pairs of tiles on their way: AT_STAGES - 1 ahead of the one in hand. A head's tiles of a page are contiguous; lanes hold the next 32 pages of the slot
        const uint32_t ring = smem_at(at_raw) + (uint32_t) (warp * AT_STAGES * PAIR + 16 * lane);
        const int tiles_log2 = c.page_log2 - 4, tile_mask = (1 << tiles_log2) - 1;
        int next = 2 * (sp.lo + t0), pages_from = next >> tiles_log2, my_page = page_at(c, q.slot, (pages_from + lane) << c.page_log2), fill = 0, use = 0;
        const int end_tile = 2 * (sp.lo + t1);
        PairSrc src;
        uint32_t there = 0;                                        // two bits a pair that was asked for: which of its tiles have a page. The newest lowest
        const auto turn_page = [&]() {
            const int pi = next >> tiles_log2;
            if (pi - pages_from >= 31) { pages_from = pi; my_page = page_at(c, q.slot, (pi + lane) << c.page_log2); }
            const int page_a = __shfl_sync(0xffffffffu, my_page, pi - pages_from);
            src.bytes_a = page_a >= 0 ? 16 : 0;
            src.a = c.pool + (page_a >= 0 ? tile_offset(c, page_a, head, next << 4, TILE) : 0) + 16 * lane;
            if (tile_mask == 0) {                                  // pages of one tile
                const int page_b = __shfl_sync(0xffffffffu, my_page, pi + 1 - pages_from);
                src.bytes_b = page_b >= 0 ? 16 : 0;
                src.b = c.pool + (page_b >= 0 ? tile_offset(c, page_b, head, 0, TILE) - TILE : 0) + 16 * lane;
                const bool first = lane < TILE % 512 / 16;
                src.mid = first ? src.a : src.b; src.bytes_mid = first ? src.bytes_a : src.bytes_b;
            } else { src.mid = src.b = src.a; src.bytes_mid = src.bytes_b = src.bytes_a; }
        };
        const auto fetch = [&]() {
            there <<= 2;
            if (next < end_tile) {
                if ((next & tile_mask) == 0) turn_page();
                copy_pair<HD>(ring + fill, src, lane);
                there |= (uint32_t) (src.bytes_a >> 4 | src.bytes_b >> 3);
                src.a += PAIR; src.mid += PAIR; src.b += PAIR;
                fill = fill == (AT_STAGES - 1) * PAIR ? 0 : fill + PAIR;
                next += 2;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        __syncwarp();                                              // nobody still reads the ring for the piece before
        turn_page();
#pragma unroll
        for (int i = 0; i < AT_STAGES - 1; i++) fetch();
        // columns: B operand of K Q^T. Lane (g, tq) holds column g's dims 32 b + 8 tq .. + 7 as pairs (n, n + 4)
        uint32_t qf[NT][NB][4];
        float factor[NT][2], offset[NB][2] = {};
        int p_hi[NT][2];                                           // last position that the lane's two columns of S^T see; -1: no column
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float v[NB][8], top = 0.f;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 8; j++) { v[b][j] = to_f(raw[n][b].v[j]); top = fmaxf(top, fabsf(v[b][j])); }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float up = top > 0.f ? query_scale(top) : 1.f;           // (a quotient by 2^126 takes the slow way of divisions, and columns without a query would)
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float by = FOLD && (j & 1) ? up * 0.0625f : up;      // 16 c is what pairs 1 and 3 of a word give
                    qf[n][b][j] = as_u(__floats2half2_rn(v[b][j] * by, v[b][j + 4] * by));
                }
            if (FOLD) {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    float sum = 0.f;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float2 x = __half22float2(as_h2(qf[n][b][j]));
                        sum = fmaf(j & 1 ? -1152.f : -1032.f, x.x + x.y, sum);      // 1024 + 8, 1024 + 16 x 8
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    offset[b][0] = __shfl_sync(0xffffffffu, sum, 8 * tq);
                    offset[b][1] = __shfl_sync(0xffffffffu, sum, 8 * tq + 4);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int cc = ct * COLS + 8 * n + 2 * tq + j;
                factor[n][j] = a.scale_log2 / __shfl_sync(0xffffffffu, up, (2 * tq + j) * 4);
                p_hi[n][j] = cc / a.group < q.count ? q.held + cc / a.group : -1;
            }
        }
        const int row_lo = ct * COLS / a.group, row_hi = min(q.count - 1, (ct * COLS + COLS - 1) / a.group);
        const int all_see_hi = q.held + row_lo, all_see_lo = a.window > 0 ? q.held + row_hi - a.window + 1 : 0;   // positions that every column sees
        float o[NT][2 * NB][4], m[NT][2], l[NT][2], base[NT][2], limit[NT][2];       // m: the largest score less P_LIFT; base: what is taken off scores, m or 0; limit: where they move
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < 2; j++) { m[n][j] = limit[n][j] = -INFINITY; l[n][j] = base[n][j] = 0.f; }
#pragma unroll
            for (int k = 0; k < 2 * NB; k++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[n][k][j] = 0.f;
        }
#pragma unroll 1
        for (int t = t0; t < t1; t++) {
            asm volatile("cp.async.wait_group %0;" :: "n"(AT_STAGES - 2) : "memory");
            __syncwarp();                                          // all lanes' copies of pair t are there, and all are done with pair t - 1
            fetch();
            const uint8_t * pair = at_raw + warp * AT_STAGES * PAIR + use;
            use = use == (AT_STAGES - 1) * PAIR ? 0 : use + PAIR;
            const uint32_t both = there >> 2 * (AT_STAGES - 1) & 3;
            if (both == 0) continue;
            const int pos = (sp.lo + t) << 5;
            float st[2][NT][4];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint8_t * tile = pair + u * TILE;
                uint32_t kw[2][NB];
                __half2 ks[2][NB / 2];
                if constexpr (NB == 4) {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint4 x = reinterpret_cast<const uint4 *>(tile)[j * 32 + lane];
                        kw[j][0] = x.x; kw[j][1] = x.y; kw[j][2] = x.z; kw[j][3] = x.w;
                    }
                    const uint4 x = reinterpret_cast<const uint4 *>(tile + 16 * HD)[g];
                    ks[0][0] = as_h2(x.x); ks[0][1] = as_h2(x.y); ks[1][0] = as_h2(x.z); ks[1][1] = as_h2(x.w);
                } else {
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint2 x = reinterpret_cast<const uint2 *>(tile)[j * 32 + lane];
                        kw[j][0] = x.x; kw[j][1] = x.y;
                    }
                    const uint2 x = reinterpret_cast<const uint2 *>(tile + 16 * HD)[g];
                    ks[0][0] = as_h2(x.x); ks[1][0] = as_h2(x.y);
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) st[u][n][j] = 0.f;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint32_t p0[4], p1[4];
                    if (FOLD) { codes8_raw(kw[0][b], p0); codes8_raw(kw[1][b], p1); }
                    else { codes8(kw[0][b], p0); codes8(kw[1][b], p1); }
                    const float d0 = b & 1 ? __high2float(ks[0][b / 2]) : __low2float(ks[0][b / 2]), d1 = b & 1 ? __high2float(ks[1][b / 2]) : __low2float(ks[1][b / 2]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float acc[4];
                        const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
                        mma_16816(acc, a0, qf[n][b][0], qf[n][b][1], offset[b]);
                        mma_16816(acc, a1, qf[n][b][2], qf[n][b][3]);
                        st[u][n][0] = fmaf(acc[0], d0, st[u][n][0]); st[u][n][1] = fmaf(acc[1], d0, st[u][n][1]);
                        st[u][n][2] = fmaf(acc[2], d1, st[u][n][2]); st[u][n][3] = fmaf(acc[3], d1, st[u][n][3]);
                    }
                }
            }
            bool more = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) { st[0][n][j] *= factor[n][j & 1]; st[1][n][j] *= factor[n][j & 1]; }
            // rows of S^T: tokens c + 4 (2 j + e) with g = 2 c + e
            if (pos + 31 > all_see_hi || pos < all_see_lo || both != 3) {
                const int p0 = pos + (g >> 1) + 4 * (g & 1);
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int p = p0 + 16 * u + 8 * (j >> 1), top = p_hi[n][j & 1];
                            if (p > top || (a.window > 0 && p <= top - a.window) || !(both >> u & 1)) st[u][n][j] = -INFINITY;
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
                        const float top = fmaxf(m[n][j], x - P_LIFT), down = top > m[n][j] ? exp2_fast(m[n][j] - top) : 1.f;
                        m[n][j] = top;
                        base[n][j] = top == -INFINITY ? 0.f : top;
                        limit[n][j] = top + (P_LIFT + P_PASS);
                        l[n][j] *= down;
#pragma unroll
                        for (int k = 0; k < 2 * NB; k++) { o[n][k][j] *= down; o[n][k][j + 2] *= down; }
                    }
            }
            uint32_t pb[2][NT][2];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        st[u][n][j] = exp2_fast(st[u][n][j] - base[n][j & 1]);
                        l[n][j & 1] += st[u][n][j];
                    }
                    pb[u][n][0] = transposed(as_u(__floats2half2_rn(st[u][n][0], st[u][n][1])));
                    pb[u][n][1] = transposed(as_u(__floats2half2_rn(st[u][n][2], st[u][n][3])));
                }
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint8_t * tile = pair + u * TILE;
#pragma unroll
                for (int bb = 0; bb < NB / 2; bb++) {
                    const uint4 y = reinterpret_cast<const uint4 *>(tile + 8 * HD)[bb * 32 + lane], z = reinterpret_cast<const uint4 *>(tile + 17 * HD)[(NB / 2) * tq + bb];
                    const uint32_t vw[2][2] = {{y.x, y.y}, {y.z, y.w}};
                    const __half2 vs[2][2] = {{as_h2(z.x), as_h2(z.y)}, {as_h2(z.z), as_h2(z.w)}};
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int b = 2 * bb + e;
                        uint32_t p0[4], p1[4];
                        codes8(vw[e][0], p0);
                        codes8(vw[e][1], p1);
#pragma unroll
                        for (int i = 0; i < 4; i++) { p0[i] = as_u(__hmul2(as_h2(p0[i]), vs[e][0])); p1[i] = as_u(__hmul2(as_h2(p1[i]), vs[e][1])); }
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const uint32_t av[4] = {p0[2 * k], p0[2 * k + 1], p1[2 * k], p1[2 * k + 1]};
#pragma unroll
                            for (int n = 0; n < NT; n++) mma_16816(o[n][2 * b + k], av, pb[u][n][0], pb[u][n][1]);
                        }
                    }
                }
            }
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
        const bool whole = t0 == 0 && t1 == sp.n;
        const size_t slot = 2 * (size_t) me + (t0 == 0 ? 1 : 0);
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int in_tile = 8 * n + 2 * tq + j, col = ct * COLS + in_tile, i = col / a.group, h = head * a.group + col - i * a.group;
                if (i >= q.count) continue;
                if (whole) {
                    const float inv = l[n][j] != 0.f ? 1.f / l[n][j] : 0.f;
                    T * y = static_cast<T *>(a.out) + ((size_t) (q.begin + i) * c.n_kv * a.group + h) * HD + 4 * g;
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        Four<T> f;
                        f.v[0] = from_f<T>(o[n][2 * b][j] * inv); f.v[1] = from_f<T>(o[n][2 * b][j + 2] * inv);
                        f.v[2] = from_f<T>(o[n][2 * b + 1][j] * inv); f.v[3] = from_f<T>(o[n][2 * b + 1][j + 2] * inv);
                        *reinterpret_cast<Four<T> *>(y + 32 * b) = f;
                    }
                } else {
                    float * y = a.part + (slot * COLS + in_tile) * HD + 4 * g;
#pragma unroll
                    for (int b = 0; b < NB; b++) *reinterpret_cast<float4 *>(y + 32 * b) = make_float4(o[n][2 * b][j], o[n][2 * b][j + 2], o[n][2 * b + 1][j], o[n][2 * b + 1][j + 2]);
                    if (g == 0) *reinterpret_cast<float2 *>(a.ml + (slot * COLS + in_tile) * 2) = make_float2(m[n][j], l[n][j]);
                }
            }
    }
}

// AJ_WARPS warps a row and head (one: eight of them a block): add the partial results of a unit that several warps shared. A warp takes every AJ_WARPS-th part, eight of them on their way at a
// time. It stands ready behind
// the kernel in front (programmatic launch): 3 to 5 us of latency behind that one's end
template <int HD, int NT, typename T, int AJ_WARPS>
__global__ void __launch_bounds__(AJ_WARPS == 1 ? 256 : AJ_WARPS * 32) k_kv4_join(const AttendArgs a) {
    constexpr int COLS = 8 * NT, E = HD / 32, BATCH = 8;
    const Cache & c = a.c;
    const int lane = threadIdx.x & 31, warp = AJ_WARPS == 1 ? 0 : threadIdx.x >> 5, n_head = c.n_kv * a.group, item = AJ_WARPS == 1 ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    const int row = item / n_head, h = item - row * n_head;
    const int s = seq_of_row_warp(c, min(row, c.n_rows - 1)), begin = min(max(c.first[max(s, 0)], 0), c.n_rows), count = min(max(c.first[max(s, 0) + 1], begin), c.n_rows) - begin;
    const int head = h / a.group, col = (row - begin) * a.group + h - head * a.group, ct = col / COLS, in_tile = col - ct * COLS;
    // every block waits, those without work too: this kernel's end is the next one's beginning, and the kernel in front still writes the workspace
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row >= c.n_rows || s < 0) return;
    const long long b0 = a.before[s], b1 = a.before[s + 1];
    const int per = (int) a.before[c.n_seq + 1], len = (int) quotient(b1 - b0, (count * a.group + COLS - 1) / COLS * c.n_kv);
    const long long u0 = b0 + (long long) (ct * c.n_kv + head) * len;
    const int w0 = (int) quotient(u0 + AT_OVER, per), w1 = (int) quotient(u0 + len - 1, per);
    if (w0 == w1) return;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.f;
    for (int w = w0 + warp; w <= w1; w += AJ_WARPS * BATCH) {
        float2 ml[BATCH];
        float x[BATCH][E];
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            const int at = w + i * AJ_WARPS;
            ml[i] = make_float2(-INFINITY, 0.f);
            const size_t slot = (2 * (size_t) at + (at == w0 ? 1 : 0)) * COLS + in_tile;
#pragma unroll
            for (int e = 0; e < E; e++) x[i][e] = 0.f;
            if (at <= w1) {
                ml[i] = *reinterpret_cast<const float2 *>(a.ml + slot * 2);
                if constexpr (E == 4) { const float4 v = *reinterpret_cast<const float4 *>(a.part + slot * HD + 4 * lane); x[i][0] = v.x; x[i][1] = v.y; x[i][2] = v.z; x[i][3] = v.w; }
                else { const float2 v = *reinterpret_cast<const float2 *>(a.part + slot * HD + 2 * lane); x[i][0] = v.x; x[i][1] = v.y; }
            }
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < BATCH; i++) top = fmaxf(top, ml[i].x);
        const float base = top == -INFINITY ? 0.f : top, old = exp2_fast(m - base);
        l *= old;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] *= old;
#pragma unroll
        for (int i = 0; i < BATCH; i++) {
            const float by = exp2_fast(ml[i].x - base);
            l = fmaf(ml[i].y, by, l);
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = fmaf(x[i][e], by, o[e]);
        }
        m = top;
    }
    if constexpr (AJ_WARPS == 1) {
        struct alignas(E * sizeof(T)) Dims { T v[E]; } y;
#pragma unroll
        for (int e = 0; e < E; e++) y.v[e] = from_f<T>(l != 0.f ? o[e] / l : 0.f);
        *reinterpret_cast<Dims *>(static_cast<T *>(a.out) + ((size_t) row * n_head + h) * HD + E * lane) = y;
    } else {
        __shared__ float sums[AJ_WARPS][HD], ml_s[AJ_WARPS][2];
#pragma unroll
        for (int e = 0; e < E; e++) sums[warp][E * lane + e] = o[e];
        if (lane == 0) { ml_s[warp][0] = m; ml_s[warp][1] = l; }
        __syncthreads();
        if (threadIdx.x < HD) {
            float top = -INFINITY, total = 0.f, y = 0.f;
#pragma unroll
            for (int i = 0; i < AJ_WARPS; i++) top = fmaxf(top, ml_s[i][0]);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int i = 0; i < AJ_WARPS; i++) {
                const float by = exp2_fast(ml_s[i][0] - base);
                total = fmaf(ml_s[i][1], by, total);
                y = fmaf(sums[i][threadIdx.x], by, y);
            }
            static_cast<T *>(a.out)[((size_t) row * n_head + h) * HD + threadIdx.x] = from_f<T>(total != 0.f ? y / total : 0.f);
        }
    }
}

}  // namespace srv
}  // namespace b200
