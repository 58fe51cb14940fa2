// kv8_attention.cu - causal attention of a ragged batch over the paged 8-bit
// KV cache (sm_100a).
//
// Row i of sequence s stands at position P = lens[s] + i and attends to the
// positions 0 .. P of its pages (its own key and value are in the cache):
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q.k_t - max),
//   k_t = ks * kq_t,  v_t = vs * vq_t
// in one pass with the running maximum and sum of the softmax.  q is rotated
// by its position here.  The reference's per-head loop (src/core/layer.rs:
// 175-333) is the same formula over one sequence's contiguous f32 cache.
//
// One warp per (row, query head): lane = D/32 dims, one token at a time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attention_core.cuh"
#include "kv8.cuh"

namespace llmrs {

namespace {

__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

template <class T, int D>
__global__ void __launch_bounds__(128) kv8_attention_kernel(Kv8Attn a)
{
    constexpr int DL = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x, h = blockIdx.y * 4 + warp;
    if (h >= a.n_heads)
        return;
    int s = -1, r0 = 0, n = 0, len = 0;
    for (int i = 0; i < a.b.n_seqs; i++) {
        kv8_seq(a.b, i, a.err, r0, n, len);
        if (n && row >= r0 && row < r0 + n) {
            s = i;
            break;
        }
    }
    if (s < 0)
        return;
    const int pos = len + row - r0, g = h / (a.n_heads / a.c.n_kv);
    const T *qp = reinterpret_cast<const T *>(a.q) + (size_t)row * a.ld_q + (size_t)h * D + lane * DL;
    float q[DL], c[DL], sn[DL], acc[DL];
#pragma unroll
    for (int k = 0; k < DL; k++) {
        q[k] = (float)qp[k];
        acc[k] = 0.0f;
    }
    if (a.r.cos) {
        rope_table_lane<D>(c, sn, lane, a.r.cos + (size_t)pos * (D / 2), a.r.sin + (size_t)pos * (D / 2));
        rope_lane<D>(q, lane, c, sn);
    }
    float m = -INFINITY, l = 0.0f;
    for (int t = 0; t <= pos; t++) {
        const int id = kv8_page(a.b, a.c, s, t / a.c.page, a.err);
        if (id < 0)
            continue;
        const size_t at = (size_t)id * a.c.n_kv + g, o = (at * a.c.page + t % a.c.page) * D + lane * DL;
        float dot = 0.0f;
#pragma unroll
        for (int k = 0; k < DL; k++)
            dot += q[k] * (float)a.c.kq[o + k];
        const float x = warp_sum(dot) * (a.c.ks[at] * a.scale);
        const float m_new = fmaxf(m, x), corr = expf(m - m_new), p = expf(x - m_new), vs = a.c.vs[at];
        l = l * corr + p;
#pragma unroll
        for (int k = 0; k < DL; k++)
            acc[k] = acc[k] * corr + p * vs * (float)a.c.vq[o + k];
        m = m_new;
    }
    T *out = reinterpret_cast<T *>(a.out) + (size_t)row * a.ld_out + (size_t)h * D + lane * DL;
#pragma unroll
    for (int k = 0; k < DL; k++)
        put(out + k, l == 0.0f ? 0.0f : acc[k] / l);
}

template <class T>
cudaError_t run(const Kv8Attn &a, cudaStream_t stream)
{
    const dim3 grid((unsigned)a.b.n_rows, (unsigned)((a.n_heads + 3) / 4));
    return a.c.D == 128 ? launch(kv8_attention_kernel<T, 128>, grid, dim3(128), 0, stream, false, a)
                        : launch(kv8_attention_kernel<T, 64>, grid, dim3(128), 0, stream, false, a);
}

} // namespace

size_t kv8_attention_workspace(int, int, int, int) { return 256; }

int kv8_prepare(void) { return LLMRS_OK; }

int kv8_attention(const Kv8Attn &a, void *, int, cudaStream_t stream)
{
    if (a.dtype == LLMRS_F32)
        LLMRS_CUDA_TRY(run<float>(a, stream));
    else if (a.dtype == LLMRS_BF16)
        LLMRS_CUDA_TRY(run<__nv_bfloat16>(a, stream));
    else
        LLMRS_CUDA_TRY(run<__half>(a, stream));
    return LLMRS_OK;
}

} // namespace llmrs
