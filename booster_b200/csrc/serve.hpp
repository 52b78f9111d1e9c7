// serve.hpp — host interface of the operators of a server that runs many sequences at once (serve.cu): a cache of keys and values in 4 bits that
// sequences hold in pages, attention over it, its pages' life, and the draw of next tokens. engine.cu wraps them in the C-ABI (b200_kv4_*,
// b200_pages_*, b200_sample); arguments are device pointers, work is enqueued on the caller's stream. Functions throw std::runtime_error.
#pragma once
#include "../../include/booster_b200.h"

namespace b200 {

void    kv4_append(const b200_kv4 & c, int dtype, const void * k, int64_t k_row, int64_t k_head, const void * v, int64_t v_row, int64_t v_head);
void    kv4_read(const b200_kv4 & c, int dtype, void * k, void * v);
int64_t kv4_attention_workspace(const b200_kv4 & c, int n_head, int max_rows);
void    kv4_attention(const b200_kv4 & c, int dtype, const void * q, int64_t q_row, int64_t q_head, int n_head, float scale, int window, int max_rows, void * out, void * work, int64_t work_bytes);
void    kv4_status(int device);
void    kv4_drill(int polls);

int64_t pages_workspace(const b200_pages & p, int n);
void    pages_reserve(const b200_pages & p, const int32_t * slots, const int32_t * first, int n, int32_t * status);
void    pages_fork(const b200_pages & p, const int32_t * parents, const int32_t * children, int n, int32_t * status, void * work, int64_t work_bytes);
void    pages_free(const b200_pages & p, const int32_t * slots, int n);
void    pages_compact(const b200_pages & p, int32_t * live, void * work, int64_t work_bytes);
void    pages_copy(const b200_pages & p, const int32_t * src, const int32_t * dst, int n, int32_t * status, void * work, int64_t work_bytes);

void    sample_rows(int device, void * stream, int dtype, const void * logits, int64_t row_stride, int n_rows, int n_vocab, const float * u, const float * temperature,
                    const int32_t * top_k, const float * top_p, const float * min_p, int32_t * ids, float * logprobs);

}  // namespace b200
