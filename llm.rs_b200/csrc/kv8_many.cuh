// kv8_many.cuh - attention over the paged 8-bit cache for many rows per
// sequence (host interface; kv8_attention.cu decides when it runs).
#pragma once

#include "kv8.cuh"

namespace llmrs {

constexpr int MANY_CTAS = 160;    // most CTAs, one per SM
constexpr int MANY_MAX_REP = 128; // query heads of a KV head: a row's vectors lie in one tile

size_t kv8_many_workspace(int head_dim, int n_heads, int n_rows);
int kv8_many_prepare(void);
// the sequences with more than `many` vectors (rows x query heads) per KV head
int kv8_many(const Kv8Attn &a, int many, void *ws, int sms, cudaStream_t stream);

} // namespace llmrs
