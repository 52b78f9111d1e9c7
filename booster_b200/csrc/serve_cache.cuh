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
// the sequence that a row belongs to: the last one that begins at or before it; -1: none
__device__ __forceinline__ int seq_of_row(const Cache & c, int row) {
    int lo = 0, hi = c.n_seq;                                     // first[lo] <= row < first[hi], as far as first ascends
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (c.first[mid] <= row) lo = mid; else hi = mid; }
    return c.first[lo] <= row && row < c.first[lo + 1] ? lo : -1;
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

// codes of four entries (lowest bits first) and the scale of their block, which eight neighbouring lanes share
template <typename T> __device__ __forceinline__ uint32_t quantize4(const float (&x)[4], bool whole, float & scale) {
    float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3])), hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
#pragma unroll
    for (int m = 1; m < 8; m <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
    float d = (-lo >= hi ? lo : hi) * -0.125f;
    d = fminf(fmaxf(d, -8160.f), 8160.f);
    d = __half2float(__float2half_rn(__bfloat162float(__float2bfloat16_rn(d))));
    if (!whole || d == 0.f) { scale = 0.f; return 0x8888u; }
    scale = d;
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float q = __fdiv_rn(x[i], d);
        float r = rintf(q);
        // 24-bit entries: a quotient that was rounded to a half lies on one side of it. (n + 1/2) d has 13 bits, so the remainder is exact. Entries of 11 or 8 bits are never that near
        if (sizeof(T) == 4 && fabsf(q - truncf(q)) == 0.5f) {
            const float rest = fmaf(-q, d, x[i]);
            if (rest != 0.f) r = (rest > 0.f) == (d > 0.f) ? ceilf(q) : floorf(q);
        }
        codes |= (uint32_t) (__float2int_rn(fminf(fmaxf(r, -8.f), 7.f)) + 8) << (4 * i);
    }
    return codes;
}

// HD / 4 lanes a row and head, four entries each. Memory bounds it: rows are read once, 4.5 bits a number are written.
template <typename T, int HD>
__global__ void __launch_bounds__(256) k_kv4_append(const Cache c, const T * k, int64_t k_row, int64_t k_head, const T * v, int64_t v_row, int64_t v_head, bool whole4) {
    constexpr int LANES = HD / 4, NB = HD / 32;
    const int64_t item = ((int64_t) blockIdx.x * blockDim.x + threadIdx.x) / LANES;
    const int li = threadIdx.x % LANES;
    const bool in = item < (int64_t) c.n_rows * c.n_kv;
    const int row = in ? (int) (item / c.n_kv) : 0, head = in ? (int) (item % c.n_kv) : 0;
    const int s = in ? seq_of_row(c, row) : -1;
    int page = -1, pos = 0;
    if (s >= 0) {
        const Seq q = seq_at(c, s);
        pos = q.held + row - q.begin;
        page = page_at(c, q.slot, pos);
    }
    float xk[4] = {}, xv[4] = {};
    if (page >= 0) {
        load4(k + row * k_row + head * k_head + 4 * li, whole4, xk);
        load4(v + row * v_row + head * v_head + 4 * li, whole4, xv);
    }
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 4; i++) fine = fine && isfinite(xk[i]) && isfinite(xv[i]);
    const unsigned mine = LANES == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
    fine = (__ballot_sync(0xffffffffu, fine) & mine) == mine;
    float dk, dv;
    const uint32_t ck = quantize4<T>(xk, fine, dk), cv = quantize4<T>(xv, fine, dv);
    if (page < 0) return;
    const int t = pos & 15, tc = t & 3, ti = t >> 2, b = li >> 3, e = li & 7;
    uint8_t * tile = c.pool + tile_offset(c, page, head, pos, 18 * HD);
    reinterpret_cast<uint16_t *>(tile)[2 * ((((ti >> 1) * 8 + 2 * tc + (ti & 1)) * 4 + (e >> 1)) * NB + b) + (e & 1)] = (uint16_t) ck;
    reinterpret_cast<uint16_t *>(tile + 8 * HD)[((((b >> 1) * 8 + e) * 4 + tc) * 2 + (b & 1)) * 4 + ti] = (uint16_t) cv;
    if (e == 0) {
        reinterpret_cast<__half *>(tile + 16 * HD)[((tc * 2 + (ti & 1)) * 2 + (ti >> 1)) * NB + b] = __float2half_rn(fine ? dk : NAN);
        reinterpret_cast<__half *>(tile + 17 * HD)[(tc * NB + b) * 4 + ti] = __float2half_rn(dv);
    }
}

// the rows' positions read back: out [n_rows][n_kv][HD]; a position without a page reads 0
template <typename T, int HD>
__global__ void __launch_bounds__(256) k_kv4_read(const Cache c, T * k, T * v) {
    constexpr int LANES = HD / 4, NB = HD / 32;
    const int64_t item = ((int64_t) blockIdx.x * blockDim.x + threadIdx.x) / LANES;
    if (item >= (int64_t) c.n_rows * c.n_kv) return;
    const int li = threadIdx.x % LANES, row = (int) (item / c.n_kv), head = (int) (item % c.n_kv), s = seq_of_row(c, row);
    if (s < 0) return;
    const Seq q = seq_at(c, s);
    const int pos = q.held + row - q.begin, page = page_at(c, q.slot, pos);
    float dk = 0.f, dv = 0.f;
    uint32_t ck = 0, cv = 0;
    if (page >= 0) {
        const int t = pos & 15, tc = t & 3, ti = t >> 2, b = li >> 3, e = li & 7;
        const uint8_t * tile = c.pool + tile_offset(c, page, head, pos, 18 * HD);
        ck = reinterpret_cast<const uint16_t *>(tile)[2 * ((((ti >> 1) * 8 + 2 * tc + (ti & 1)) * 4 + (e >> 1)) * NB + b) + (e & 1)];
        cv = reinterpret_cast<const uint16_t *>(tile + 8 * HD)[((((b >> 1) * 8 + e) * 4 + tc) * 2 + (b & 1)) * 4 + ti];
        dk = __half2float(reinterpret_cast<const __half *>(tile + 16 * HD)[((tc * 2 + (ti & 1)) * 2 + (ti >> 1)) * NB + b]);
        dv = __half2float(reinterpret_cast<const __half *>(tile + 17 * HD)[(tc * NB + b) * 4 + ti]);
    }
    Four<T> fk, fv;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        fk.v[i] = from_f<T>((float) ((int) (ck >> (4 * i) & 15) - 8) * dk);
        fv.v[i] = from_f<T>((float) ((int) (cv >> (4 * i) & 15) - 8) * dv);
    }
    const size_t at = ((size_t) row * c.n_kv + head) * HD + 4 * li;
    *reinterpret_cast<Four<T> *>(k + at) = fk;
    *reinterpret_cast<Four<T> *>(v + at) = fv;
}

}  // namespace srv
}  // namespace b200
