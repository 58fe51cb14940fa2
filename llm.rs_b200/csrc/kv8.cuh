// kv8.cuh - the paged 8-bit KV cache and the operators over it (host interface),
// and the device helpers that read a ragged batch.
//
// Cache: int8 codes [page][kv head][page_size][D] with one f32 scale per (page,
// kv head); a value is code * scale.  Batch: sequence s owns the packed rows
// row_start[s] .. row_start[s+1]-1, has lens[s] tokens in the cache before
// them, and table[s][p] names the page of its positions p*page_size onwards.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.cuh"

namespace llmrs {

struct Kv8 {
    int8_t *kq, *vq;
    float *ks, *vs;
    int n_pages, page, n_kv, D;
};

struct Kv8Batch {
    const int *row_start, *lens, *table;
    int n_seqs, max_pages;
    int n_rows; // rows of the packed buffers
    int n_pos;  // positions a row may have: the page table's reach and the RoPE table's
};

// RoPE tables [n_pos][D/2]; cos == nullptr: rows are not rotated
struct Kv8Rope {
    const float *cos, *sin;
};

int kv8_append(const Kv8 &c, const Kv8Batch &b, const void *k, const void *v, int dtype, long long ld,
               const Kv8Rope &r, uint32_t *err, cudaStream_t stream);
int kv8_read(const Kv8 &c, const int *pages, int n, void *k, void *v, int dtype, uint32_t *err, cudaStream_t stream);

struct Kv8Attn {
    Kv8 c;
    Kv8Batch b;
    Kv8Rope r;
    const void *q;
    void *out;
    long long ld_q, ld_out; // elements
    int dtype, n_heads;
    float scale;            // of q.k before the softmax
    uint32_t *err;
};
size_t kv8_attention_workspace(int n_heads, int n_kv, int head_dim, int n_rows, int n_seqs);
int kv8_attention(const Kv8Attn &a, void *ws, int sms, cudaStream_t stream);
// set kernel attributes on the current device (once per context, outside capture)
int kv8_prepare(void);

#ifdef __CUDACC__

// Sequence s of the batch: first packed row, rows and cached tokens.  A
// sequence whose numbers lead outside the buffers counts as empty and sets
// the error word, so no later index needs a check but the page ids'.
__device__ __forceinline__ void kv8_seq(const Kv8Batch &b, int s, uint32_t *err, int &r0, int &n, int &len)
{
    r0 = b.row_start[s];
    const int r1 = b.row_start[s + 1];
    len = b.lens[s];
    n = r1 - r0;
    if (r0 == r1)
        return;
    if (r0 < 0 || r1 < r0 || r1 > b.n_rows || len < 0 || (long long)len + n > (long long)b.n_pos) {
        n = 0;
        atomicCAS(err, 0u, (uint32_t)DEV_ERR_BAD_BATCH);
    }
}

// page id of position block p of sequence s; -1 (and the error word) when it
// names no page of the pool
__device__ __forceinline__ int kv8_page(const Kv8Batch &b, const Kv8 &c, int s, int p, uint32_t *err)
{
    const int id = b.table[(size_t)s * b.max_pages + p];
    if (id < 0 || id >= c.n_pages) {
        atomicCAS(err, 0u, (uint32_t)DEV_ERR_BAD_PAGE);
        return -1;
    }
    return id;
}

// Whole block (NT threads): unit u of the units that the sequences own in
// order, count(s) of them each.  Returns the sequence (-1: there is no unit u)
// and the unit's index within it.  One coalesced pass of loads and one scan
// per NT sequences.
template <int NT, class Count>
__device__ __forceinline__ int kv8_find_unit(int n_seqs, long long u, Count count, long long &within)
{
    __shared__ long long s_warp[NT / 32];
    __shared__ long long s_at;
    __shared__ int s_seq;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0)
        s_seq = -1;
    long long base = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += NT) {
        const int s = s0 + threadIdx.x;
        const long long c = s < n_seqs ? count(s) : 0;
        long long x = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o)
                x += y;
        }
        if (lane == 31)
            s_warp[warp] = x;
        __syncthreads();
        long long before = base, all = base;
#pragma unroll
        for (int w = 0; w < NT / 32; w++) {
            if (w < warp)
                before += s_warp[w];
            all += s_warp[w];
        }
        const long long lo = before + x - c;
        if (u >= lo && u < lo + c) {
            s_seq = s;
            s_at = u - lo;
        }
        __syncthreads();
        if (s_seq >= 0)
            break;
        base = all;
    }
    within = s_at;
    return s_seq;
}

// four consecutive elements of a row as floats (16- or 8-byte load)
__device__ __forceinline__ float4 kv8_load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
template <class T>
__device__ __forceinline__ float4 kv8_load4(const T *p)
{
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    T h[4];
    memcpy(h, &w, 8);
    return make_float4((float)h[0], (float)h[1], (float)h[2], (float)h[3]);
}

#endif // __CUDACC__

} // namespace llmrs
