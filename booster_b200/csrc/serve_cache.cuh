// serve_cache.cuh — the paged cache of 4-bit keys and values: its layout, writing rows into it, reading them back (sm_100a).
//
// A number x of a block of 32 neighbouring entries of a head's row is held as a code c of 4 bits and stands for (c - 8) d. With lo, hi the block's smallest and largest entry,
//   e = lo where -lo >= hi, else hi;   d = e / -8, at most 8160 in magnitude, rounded to 8 significant bits (bfloat16) and stored as fp16;   c = rint(x / d) + 8 in 0 .. 15
// so the entry of largest magnitude is code 0. 8 bits of d times 4 bits of c - 8 are exact in fp16: kernels multiply what is held, not a rounding of it. 4.5 bits a number.
// A token with an infinity or a NaN in a head's key or value holds NaN as its key's scales and 0 as its value's: who sees the token answers NaN for the head, nobody else does, and
// values in the cache are always finite (a masked position's weight 0 may be multiplied with them).
//
// A tile is 16 tokens of one KV head, 18 x head_dim contiguous bytes in the order in which a warp's lane (g = lane / 4, q = lane % 4) multiplies them. Token t = c + 4 i:
//   K codes   words [i / 2][g = 2 c + i % 2][q][block]: dims 32 block + 8 q + 0 .. 7, lowest bits first
//   V codes   16-bit units [block / 2][g][c][block % 2][i]: dims 32 block + 4 g + 0 .. 3, so that a word holds 4 dims of two tokens
//   K scales  fp16 [c][i % 2][i / 2][block]
//   V scales  fp16 [c][block][i]
// A page is page_tokens / 16 tiles of every KV head: [n_head_kv][page_tokens / 16][18 head_dim].
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace b200 {
namespace srv {

struct Cache {
    uint8_t * pool;
    int64_t page_stride;                 // bytes from page to page
    int n_pages, page_log2, n_kv;        // page_tokens = 1 << page_log2
    const int32_t * table;
    int64_t table_stride;
    int n_slots, max_pages;
    const int32_t * held, * slots, * first;
    int n_seq, n_rows;
};

// a sequence of the step: rows begin .. begin + count - 1, at positions held .. held + count - 1. What tables say is bounded here, so that no kernel reads out of range by it
struct Seq { int slot, begin, count, held; };
__device__ __forceinline__ Seq seq_at(const Cache & c, int s) {
    Seq r;
    r.slot = c.slots ? c.slots[s] : s;
    r.begin = min(max(c.first[s], 0), c.n_rows);
    r.count = min(max(c.first[s + 1], r.begin), c.n_rows) - r.begin;
    if ((unsigned) r.slot >= (unsigned) c.n_slots) { r.slot = -1; r.held = 0; }
    else r.held = min(max(c.held[r.slot], 0), c.max_pages << c.page_log2);
    return r;
}
// the page of a slot's position, -1 where there is none of this pool
__device__ __forceinline__ int page_at(const Cache & c, int slot, int pos) {
    const int i = pos >> c.page_log2;
    if (slot < 0 || i >= c.max_pages) return -1;
    const int page = c.table[(int64_t) slot * c.table_stride + i];
    return (unsigned) page < (unsigned) c.n_pages ? page : -1;
}
__device__ __forceinline__ size_t tile_offset(const Cache & c, int page, int head, int pos, int tile_bytes) {
    const int tiles_log2 = c.page_log2 - 4;
    return (size_t) page * c.page_stride + (size_t) ((head << tiles_log2) + ((pos >> 4) & ((1 << tiles_log2) - 1))) * tile_bytes;
}

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// four entries in one access where `whole` says that they stand on their own alignment
template <typename T> struct alignas(4 * sizeof(T)) Four { T v[4]; };
template <typename T> struct alignas(2 * sizeof(T)) Two { T v[2]; };
template <typename T> __device__ __forceinline__ void load4(const T * p, bool whole, float (&x)[4]) {
    if (whole) {
        const Four<T> f = *reinterpret_cast<const Four<T> *>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = to_f(f.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = to_f(p[i]);
    }
}

// the larger of each side of a pair of T, a NaN where one is: (-smallest, largest) of a block go through the lanes as one word
template <typename T> __device__ __forceinline__ uint32_t pair_max(uint32_t x, uint32_t y);
template <> __device__ __forceinline__ uint32_t pair_max<__half>(uint32_t x, uint32_t y) { uint32_t r; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y)); return r; }
template <> __device__ __forceinline__ uint32_t pair_max<__nv_bfloat16>(uint32_t x, uint32_t y) { uint32_t r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y)); return r; }
__device__ __forceinline__ float max_nan(float x, float y) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y)); return r; }

// of the block of 32 that eight neighbouring lanes share: whether it is finite, and its scale
template <typename T> __device__ __forceinline__ bool block_scale(const float (&x)[4], float & d) {
    float lo = max_nan(max_nan(-x[0], -x[1]), max_nan(-x[2], -x[3])), hi = max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3]));      // lo: turned round
    if constexpr (sizeof(T) == 2) {
        Two<T> p = {{from_f<T>(lo), from_f<T>(hi)}};                      // (entries of T: exact)
        uint32_t w = *reinterpret_cast<uint32_t *>(&p);
#pragma unroll
        for (int m = 1; m < 8; m <<= 1) w = pair_max<T>(w, __shfl_xor_sync(0xffffffffu, w, m));
        p = *reinterpret_cast<Two<T> *>(&w);
        lo = to_f(p.v[0]); hi = to_f(p.v[1]);
    } else {
#pragma unroll
        for (int m = 1; m < 8; m <<= 1) {
            lo = max_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
        }
    }
    d = (lo >= hi ? -lo : hi) * -0.125f;
    d = fminf(fmaxf(d, -8160.f), 8160.f);
    d = __half2float(__float2half_rn(__bfloat162float(__float2bfloat16_rn(d)))) + 0.f;
    return lo < INFINITY && hi < INFINITY;
}
// codes of four entries of a block of scale d, lowest bits first
template <typename T> __device__ __forceinline__ uint32_t codes4(const float (&x)[4], float d) {
    const float by = __fdividef(1.f, d);
    float c[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 2) {
            // rint(x / d): the quotient, put right by its remainder, is exact where x / d is a half, and no other quotient of 11 and 8 bits is as near to one as its rounding
            const float q = x[i] * by, r = fmaf(fmaf(-q, d, x[i]), by, q);
            c[i] = fminf(fmaxf(r, -8.f), 7.f) + 12582912.f - 12582912.f;       // 1.5 x 2^23: rounds to a whole number
        } else {
            // with 24 bits a quotient may round to a half that it is not. The remainder of the nearest code tells the neighbour: where it is about d / 2 it is exact
            const float half = 0.5f * fabsf(d), t = fmaf(x[i], by, 12582912.f), rest = fmaf(-(t - 12582912.f), d, x[i]);
            c[i] = t - 12582912.f;
            if (fabsf(rest) > half || (fabsf(rest) == half && (__float_as_int(t) & 1))) c[i] += (rest > 0.f) == (d > 0.f) ? 1.f : -1.f;
            c[i] = fminf(fmaxf(c[i], -8.f), 7.f);
        }
    }
    // c0 + 16 c1 + 256 c2 + 4096 c3 + 8 x 0x1111, below 2^16, as last bits
    const uint32_t w = __float_as_uint(fmaf(c[3], 4096.f, fmaf(c[2], 256.f, fmaf(c[1], 16.f, c[0]))) + (8388608.f + 34952.f)) & 0xffffu;
    return d == 0.f ? 0x8888u : w;
}

// the sequence that a row belongs to, the last one that begins at or before it, looked for by a whole warp, 32 places at a time; -1: none
__device__ __forceinline__ int seq_of_row_warp(const Cache & c, int row) {
    const int lane = threadIdx.x & 31;
    int s = 0, n = c.n_seq;
    while (n > 1) {
        const int step = (n + 31) >> 5, i = s + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, lane * step < n && c.first[min(i, c.n_seq)] <= row);
        const int k = m ? 31 - __clz(m) : 0;
        s += k * step;
        n = min(step, n - k * step);
    }
    return c.first[s] <= row && row < c.first[s + 1] ? s : -1;
}

// where a lane's four entries of token t stand in a tile: 16-bit units of K and V codes, and the scale of their block
template <int HD> __device__ __forceinline__ int k_unit(int li, int t) { return 2 * ((((t >> 3) * 8 + 2 * (t & 3) + (t >> 2 & 1)) * 4 + ((li & 7) >> 1)) * (HD / 32) + (li >> 3)) + (li & 1); }
template <int HD> __device__ __forceinline__ int v_unit(int li, int t) { return ((((li >> 4) * 8 + (li & 7)) * 4 + (t & 3)) * 2 + (li >> 3 & 1)) * 4 + (t >> 2); }
template <int HD> __device__ __forceinline__ int k_scale_at(int li, int t) { return (((t & 3) * 2 + (t >> 2 & 1)) * 2 + (t >> 3)) * (HD / 32) + (li >> 3); }
template <int HD> __device__ __forceinline__ int v_scale_at(int li, int t) { return ((t & 3) * (HD / 32) + (li >> 3)) * 4 + (t >> 2); }

template <typename T> struct RowSrc { const T * k; int64_t k_row, k_head; const T * v; int64_t v_row, v_head; bool whole4; };
// codes and scales of one row and head, HD / 4 lanes of four entries each
struct Codes { uint32_t k, v; float dk, dv; };
template <typename T, int HD> __device__ __forceinline__ Codes codes_of(const float (&xk)[4], const float (&xv)[4]) {
    Codes r;
    const bool fine_k = block_scale<T>(xk, r.dk), fine_v = block_scale<T>(xv, r.dv);
    const unsigned mine = HD == 128 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
    const bool fine = (__ballot_sync(0xffffffffu, fine_k && fine_v) & mine) == mine;
    r.k = fine ? codes4<T>(xk, r.dk) : 0x8888u;
    r.v = fine ? codes4<T>(xv, r.dv) : 0x8888u;
    if (!fine) { r.dk = NAN; r.dv = 0.f; }
    return r;
}
template <int HD> __device__ __forceinline__ void put_scales(uint8_t * tile, int li, int t, const Codes & q) {
    if ((li & 7) == 0) {
        reinterpret_cast<__half *>(tile + 16 * HD)[k_scale_at<HD>(li, t)] = __float2half_rn(q.dk);
        reinterpret_cast<__half *>(tile + 17 * HD)[v_scale_at<HD>(li, t)] = __float2half_rn(q.dv);
    }
}

// A warp a row and PASSES passes of its heads (a head at head_dim 128, two at 64), all asked for together. Latency bounds it: row -> sequence -> slot -> page, then 2 bytes a lane into the
// two halves of a tile; with thousands of rows the arithmetic of codes does (173 instructions a row and head). 48 rows of 8 heads of 128 in 4.5 us, 8192 in 19
// (43 MB, 2.2 TB/s). Warps that took whole tiles of long portions, their V codes as words, were no faster at 8192 rows of 8 heads (26.8 us written and read, 25.4 this way) and slower
// at 128 sequences of 16 rows (20.1 and 12.3); 4 x 8192 rows 88.6 and 92.8.
template <typename T, int HD, int PASSES>
__global__ void __launch_bounds__(256) k_kv4_append(const Cache c, const RowSrc<T> src, int parts) {
    constexpr int LANES = HD / 4, PER = 32 / LANES;
    const int64_t item = ((int64_t) blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31, li = lane % LANES, row = (int) (item / parts), h0 = (int) (item % parts) * PASSES * PER + lane / LANES;
    if (row >= c.n_rows) return;
    float xk[PASSES][4] = {}, xv[PASSES][4] = {};
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int head = h0 + i * PER;
        if (head < c.n_kv) {
            load4(src.k + row * src.k_row + head * src.k_head + 4 * li, src.whole4, xk[i]);
            load4(src.v + row * src.v_row + head * src.v_head + 4 * li, src.whole4, xv[i]);
        }
    }
    const int s = seq_of_row_warp(c, row);
    if (s < 0) return;
    const Seq q = seq_at(c, s);
    const int pos = q.held + row - q.begin, page = page_at(c, q.slot, pos), t = pos & 15;
    if (page < 0) return;
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const Codes r = codes_of<T, HD>(xk[i], xv[i]);
        const int head = h0 + i * PER;
        if (head < c.n_kv) {
            uint8_t * tile = c.pool + tile_offset(c, page, head, pos, 18 * HD);
            reinterpret_cast<uint16_t *>(tile)[k_unit<HD>(li, t)] = (uint16_t) r.k;
            reinterpret_cast<uint16_t *>(tile + 8 * HD)[v_unit<HD>(li, t)] = (uint16_t) r.v;
            put_scales<HD>(tile, li, t, r);
        }
        __syncwarp();
    }
}

template <typename T> __device__ __forceinline__ Four<T> held_values(uint32_t codes, float d) {
    Four<T> f;
#pragma unroll
    for (int i = 0; i < 4; i++) f.v[i] = from_f<T>((float) ((int) (codes >> (4 * i) & 15) - 8) * d);
    return f;
}
// the rows' positions read back: out [n_rows][n_kv][HD]; a position without a page reads 0. As above; 8192 rows in 9 us (4.6 TB/s)
template <typename T, int HD, int PASSES>
__global__ void __launch_bounds__(256) k_kv4_read(const Cache c, T * k, T * v, int parts) {
    constexpr int LANES = HD / 4, PER = 32 / LANES;
    const int64_t item = ((int64_t) blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31, li = lane % LANES, row = (int) (item / parts), h0 = (int) (item % parts) * PASSES * PER + lane / LANES;
    if (row >= c.n_rows) return;
    const int s = seq_of_row_warp(c, row);
    if (s < 0) return;
    const Seq q = seq_at(c, s);
    const int pos = q.held + row - q.begin, page = page_at(c, q.slot, pos), t = pos & 15;
    uint32_t ck[PASSES] = {}, cv[PASSES] = {};
    float dk[PASSES] = {}, dv[PASSES] = {};
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int head = h0 + i * PER;
        if (page >= 0 && head < c.n_kv) {
            const uint8_t * tile = c.pool + tile_offset(c, page, head, pos, 18 * HD);
            ck[i] = reinterpret_cast<const uint16_t *>(tile)[k_unit<HD>(li, t)];
            cv[i] = reinterpret_cast<const uint16_t *>(tile + 8 * HD)[v_unit<HD>(li, t)];
            dk[i] = __half2float(reinterpret_cast<const __half *>(tile + 16 * HD)[k_scale_at<HD>(li, t)]);
            dv[i] = __half2float(reinterpret_cast<const __half *>(tile + 17 * HD)[v_scale_at<HD>(li, t)]);
        }
    }
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int head = h0 + i * PER;
        if (head < c.n_kv) {
            const size_t at = ((size_t) row * c.n_kv + head) * HD + 4 * li;
            *reinterpret_cast<Four<T> *>(k + at) = held_values<T>(ck[i], dk[i]);
            *reinterpret_cast<Four<T> *>(v + at) = held_values<T>(cv[i], dv[i]);
        }
    }
}
}  // namespace srv
}  // namespace b200
