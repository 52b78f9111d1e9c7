// serve_attn.cuh — attention of a step's rows over the 4-bit cache (sm_100a): few rows of many sequences.
//
// A unit of work is a sequence's columns (a column is a row and a query head of one KV head: 8 NT of them) over the tiles of 16 tokens that its rows see. All units' tiles stand in one
// line, which is cut evenly over all warps of the grid: a warp walks its piece by itself, with the running maximum and sum of the soft-max in registers, and ends a unit that others share
// with a partial result that k_kv4_join adds. So sequences of any lengths fill the card, and nothing is waited for inside.
//   S^T = K Q^T: a tile's codes are the A operand of mma.sync (16 tokens x 16 dims), the columns the B operand. A block's 32 products are summed as codes and scaled once.
//   O^T += V^T P^T: V's codes times their scales (exact in fp16) are the A operand (16 dims x 16 tokens); P^T comes from S^T by movmatrix.
// P is rounded to fp16 (2^-11), the one rounding beside the output's; q is scaled by a power of two into fp16's range, which keeps its bits. Sums are fp32.
#pragma once
#include "serve_cache.cuh"

namespace b200 {
namespace srv {

struct AttendArgs {
    Cache c;
    const void * q;
    int64_t q_row, q_head;
    void * out;                          // [n_rows][n_head][HD]
    int group, col_tiles_max;
    float scale_log2;                    // scale x log2(e)
    int window;                          // 0: all positions
    // workspace
    long long * before;                  // [n_seq + 1] tiles in front of each sequence; [n_seq + 1]: tiles of a warp
    float * part, * ml;                  // [2 x warps][8 NT][HD], [2 x warps][8 NT][2]
};

constexpr int AT_WARPS = 8, AT_MAX_SEQ = 4096;

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) { uint32_t r; asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x)); return r; }
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<__half2 *>(&x); }
__device__ __forceinline__ uint32_t as_u(__half2 x) { return *reinterpret_cast<uint32_t *>(&x); }
__device__ __forceinline__ float exp2_fast(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// the eight codes of a word less 8, as pairs (n, n + 4) of nibbles: 1024 + c and 1024 + 16 c are fp16 numbers with the code in their last bits
__device__ __forceinline__ void codes8(uint32_t w, uint32_t (&p)[4]) {
    const __half2 eight = as_h2(0xe408e408u), sixteenth = as_h2(0x2c002c00u), seventy_two = as_h2(0xd480d480u);   // -1032, 1 / 16, -72
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t x = i ? w >> 8 : w;
        p[2 * i] = as_u(__hadd2(as_h2((x & 0x000f000fu) | 0x64006400u), eight));
        p[2 * i + 1] = as_u(__hfma2(as_h2((x & 0x00f000f0u) | 0x64006400u), sixteenth, seventy_two));
    }
}

// tiles [t_lo, t_lo + n) that the rows a .. b of a sequence see, one at least (it may have nothing to see in it)
struct Span { int lo, n; };
__device__ __forceinline__ Span span_of(const Cache & c, const Seq & q, int window, int a, int b) {
    const int last = min(q.held + b, (c.max_pages << c.page_log2) - 1);
    const int first = window > 0 ? max(0, q.held + a - window + 1) : 0;
    Span s;
    s.lo = first >> 4;
    s.n = q.slot < 0 || last < first ? 1 : (last >> 4) - s.lo + 1;
    return s;
}
// a sequence's units: column tiles x KV heads, of which each column tile has a span of its own. Units of a sequence are made equally long: the span of all its rows
__device__ __forceinline__ int col_tiles(const Seq & q, int group, int cols) { return (q.count * group + cols - 1) / cols; }

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(AT_WARPS * 32) k_kv4_attend(const AttendArgs a) {
    constexpr int NB = HD / 32, COLS = 8 * NT, TILE = 18 * HD;
    extern __shared__ long long before[];                          // [n_seq + 1]
    __shared__ long long sums[AT_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3;
    const Cache & c = a.c;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // tiles in front of each sequence
    {
        const int each = (c.n_seq + AT_WARPS * 32 - 1) / (AT_WARPS * 32), s0 = min(c.n_seq, tid * each), s1 = min(c.n_seq, s0 + each);
        long long mine = 0;
        for (int s = s0; s < s1; s++) {
            const Seq q = seq_at(c, s);
            before[s] = mine;
            mine += q.count ? (long long) col_tiles(q, a.group, COLS) * c.n_kv * span_of(c, q, a.window, 0, q.count - 1).n : 0;
        }
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
    const long long per = max(1ll, (total + n_warps - 1) / n_warps);
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
        const Span sp = span_of(c, q, a.window, 0, q.count - 1);
        const int x = (int) (at - before[s]), unit = x / sp.n, t0 = x - unit * sp.n, t1 = (int) min((long long) sp.n, t0 + (end - at));
        const int ct = unit / c.n_kv, head = unit - ct * c.n_kv;
        at += t1 - t0;
        // columns: B operand of K Q^T. Lane (g, tq) holds column g's dims 32 b + 8 tq .. + 7 as pairs (n, n + 4)
        uint32_t qf[NT][NB][4];
        float factor[NT][2];
        int p_hi[NT][2];                                           // last position that the lane's two columns of S^T see; -1: no column
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int col = ct * COLS + 8 * n + g, i = col / a.group, h = head * a.group + col - i * a.group;
            const bool in = i < q.count;
            float v[NB][8], top = 0.f;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    v[b][j] = in ? to_f(static_cast<const T *>(a.q)[(q.begin + i) * a.q_row + h * a.q_head + 32 * b + 8 * tq + j]) : 0.f;
                    top = fmaxf(top, fabsf(v[b][j]));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // a power of two that brings the column's largest entry to 2^13 .. 2^14
            const int e = min(126, max(-126, 140 - (int) (__float_as_uint(top) >> 23)));
            const float up = top > 0.f && top < INFINITY ? __uint_as_float((uint32_t) (127 + e) << 23) : 1.f;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int j = 0; j < 4; j++) qf[n][b][j] = as_u(__floats2half2_rn(v[b][j] * up, v[b][j + 4] * up));
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int cc = ct * COLS + 8 * n + 2 * tq + j;
                factor[n][j] = a.scale_log2 / __shfl_sync(0xffffffffu, up, (2 * tq + j) * 4);
                p_hi[n][j] = cc / a.group < q.count ? q.held + cc / a.group : -1;
            }
        }
        const int row_lo = ct * COLS / a.group, row_hi = min(q.count - 1, (ct * COLS + COLS - 1) / a.group);
        const int all_see_hi = q.held + row_lo, all_see_lo = a.window > 0 ? q.held + row_hi - a.window + 1 : 0;   // positions that every column sees
        float o[NT][2 * NB][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < 2; j++) { m[n][j] = -INFINITY; l[n][j] = 0.f; }
#pragma unroll
            for (int k = 0; k < 2 * NB; k++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[n][k][j] = 0.f;
        }
#pragma unroll 1
        for (int t = t0; t < t1; t++) {
            const int pos = (sp.lo + t) << 4, page = page_at(c, q.slot, pos);
            if (page < 0) continue;
            const uint8_t * tile = c.pool + tile_offset(c, page, head, pos, TILE);
            uint32_t kw[2][NB], vw[NB][2];
            __half ks[2][NB];
            __half2 vs[NB][2];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    kw[j][b] = reinterpret_cast<const uint32_t *>(tile)[(j * 32 + lane) * NB + b];
                    vw[b][j] = reinterpret_cast<const uint32_t *>(tile + 8 * HD)[((b >> 1) * 32 + lane) * 4 + (b & 1) * 2 + j];
                    ks[j][b] = reinterpret_cast<const __half *>(tile + 16 * HD)[(g * 2 + j) * NB + b];
                    vs[b][j] = reinterpret_cast<const __half2 *>(tile + 17 * HD)[(tq * NB + b) * 2 + j];
                }
            float st[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) st[n][j] = 0.f;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint32_t p0[4], p1[4];
                codes8(kw[0][b], p0);
                codes8(kw[1][b], p1);
                const float d0 = __half2float(ks[0][b]), d1 = __half2float(ks[1][b]);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                    const uint32_t a0[4] = {p0[0], p1[0], p0[1], p1[1]}, a1[4] = {p0[2], p1[2], p0[3], p1[3]};
                    mma_16816(acc, a0, qf[n][b][0], qf[n][b][1]);
                    mma_16816(acc, a1, qf[n][b][2], qf[n][b][3]);
                    st[n][0] = fmaf(acc[0], d0, st[n][0]); st[n][1] = fmaf(acc[1], d0, st[n][1]);
                    st[n][2] = fmaf(acc[2], d1, st[n][2]); st[n][3] = fmaf(acc[3], d1, st[n][3]);
                }
            }
            // rows of S^T: tokens c + 4 (2 j + e) with g = 2 c + e
            const bool edge = pos + 15 > all_see_hi || pos < all_see_lo || row_hi < 0;
            const int p0 = pos + (g >> 1) + 4 * (g & 1);
            bool more = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    st[n][j] *= factor[n][j & 1];
                    if (edge) {
                        const int p = p0 + 8 * (j >> 1), top = p_hi[n][j & 1];
                        if (p > top || (a.window > 0 && p <= top - a.window)) st[n][j] = -INFINITY;
                    }
                    more = more || st[n][j] > m[n][j & 1] + 8.f;
                }
            // the maximum moves only when a score passes it by 2^8: P stays in fp16's range below that
            if (__any_sync(0xffffffffu, more)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float x = fmaxf(st[n][j], st[n][j + 2]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        const float top = fmaxf(m[n][j], x), down = top > m[n][j] ? exp2_fast(m[n][j] - top) : 1.f;
                        m[n][j] = top;
                        l[n][j] *= down;
#pragma unroll
                        for (int k = 0; k < 2 * NB; k++) { o[n][k][j] *= down; o[n][k][j + 2] *= down; }
                    }
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float base = m[n][j & 1] == -INFINITY ? 0.f : m[n][j & 1];
                    st[n][j] = exp2_fast(st[n][j] - base);
                    l[n][j & 1] += st[n][j];
                }
                pb[n][0] = transposed(as_u(__floats2half2_rn(st[n][0], st[n][1])));
                pb[n][1] = transposed(as_u(__floats2half2_rn(st[n][2], st[n][3])));
            }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint32_t p0[4], p1[4];
                codes8(vw[b][0], p0);
                codes8(vw[b][1], p1);
#pragma unroll
                for (int i = 0; i < 4; i++) { p0[i] = as_u(__hmul2(as_h2(p0[i]), vs[b][0])); p1[i] = as_u(__hmul2(as_h2(p1[i]), vs[b][1])); }
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t av[4] = {p0[2 * k], p0[2 * k + 1], p1[2 * k], p1[2 * k + 1]};
#pragma unroll
                    for (int n = 0; n < NT; n++) mma_16816(o[n][2 * b + k], av, pb[n][0], pb[n][1]);
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

// a warp a row and head: adds the partial results of a unit that several warps shared, in their order
template <int HD, int NT, typename T>
__global__ void __launch_bounds__(256) k_kv4_join(const AttendArgs a) {
    constexpr int COLS = 8 * NT, E = HD / 32;
    const Cache & c = a.c;
    const int lane = threadIdx.x & 31, n_head = c.n_kv * a.group;
    const int64_t item = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (item >= (int64_t) c.n_rows * n_head) return;
    const int row = (int) (item / n_head), h = (int) (item % n_head), s = seq_of_row(c, row);
    if (s < 0) return;
    const int begin = min(max(c.first[s], 0), c.n_rows), count = min(max(c.first[s + 1], begin), c.n_rows) - begin;
    const int head = h / a.group, col = (row - begin) * a.group + h - head * a.group, ct = col / COLS, in_tile = col - ct * COLS;
    const long long b0 = a.before[s], per = a.before[c.n_seq + 1];
    const int n = (int) ((a.before[s + 1] - b0) / ((long long) ((count * a.group + COLS - 1) / COLS) * c.n_kv));
    const long long u0 = b0 + (long long) (ct * c.n_kv + head) * n, w0 = u0 / per, w1 = (u0 + n - 1) / per;
    if (w0 == w1) return;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.f;
    for (long long w = w0; w <= w1; w++) {
        const size_t slot = 2 * (size_t) w + (w == w0 ? 1 : 0);
        const float2 ml = *reinterpret_cast<const float2 *>(a.ml + (slot * COLS + in_tile) * 2);
        const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.f : top, old = exp2_fast(m - base), now = exp2_fast(ml.x - base);
        l = l * old + ml.y * now;
        const float * y = a.part + (slot * COLS + in_tile) * HD + E * lane;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * old + y[e] * now;
        m = top;
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    T * y = static_cast<T *>(a.out) + ((size_t) row * n_head + h) * HD + E * lane;
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = from_f<T>(o[e] * inv);
}

}  // namespace srv
}  // namespace b200
