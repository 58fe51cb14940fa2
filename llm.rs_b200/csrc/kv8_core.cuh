// kv8_core.cuh - device pieces that both attention kernels over the paged 8-bit
// cache use: conversions, row stores, and the kernel that joins the pieces of a
// softmax.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv8.cuh"

namespace llmrs {

namespace {

// probabilities become f16 at this scale: p in [0, 1] keeps 11 bits down to
// 2^-28, and 22 bits as two pieces down to 2^-17
constexpr float P_SCALE = 16384.0f;
constexpr float P_SCALE_LOG2 = 14.0f;
constexpr int JOIN_SLOTS = 1920; // most ranges of tiles that one launch cuts
constexpr int JT = 256;          // threads of the joining kernel

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two int8 codes, offset by 128 to unsigned bytes, as f16 values: the byte
// under the exponent of 1024 is 1024 + code + 128, and the difference is exact.
__device__ __forceinline__ uint32_t codes_f16(uint32_t biased, uint32_t select)
{
    const uint32_t w = __byte_perm(biased, 0x64646464u, select);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&w), __floats2half2_rn(1152.0f, 1152.0f));
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ uint32_t pack16(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// N (a multiple of 16/sizeof(T) ... 16) consecutive floats to a row of T
template <int N>
__device__ __forceinline__ void store_row(float *p, const float (&x)[N])
{
#pragma unroll
    for (int i = 0; i < N; i += 4)
        *reinterpret_cast<float4 *>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}
template <int N>
__device__ __forceinline__ void store_row(__half *p, const float (&x)[N])
{
#pragma unroll
    for (int i = 0; i < N; i += 8)
        *reinterpret_cast<uint4 *>(p + i) = make_uint4(pack16(x[i], x[i + 1]), pack16(x[i + 2], x[i + 3]),
                                                       pack16(x[i + 4], x[i + 5]), pack16(x[i + 6], x[i + 7]));
}
template <int N>
__device__ __forceinline__ void store_row(__nv_bfloat16 *p, const float (&x)[N])
{
#pragma unroll
    for (int i = 0; i < N; i += 8) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[i + 2 * j], x[i + 2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t *>(&h);
        }
        *reinterpret_cast<uint4 *>(p + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Wait for a barrier's phase, like mbar_wait, in few instructions: a try suspends
// the warp for a while, and a million tries without the phase set the error word.
// The pause between tries leaves the issue slots to the warps at work (many-rows
// kernel: 2 %).
__device__ __forceinline__ bool kv8_wait(uint64_t *bar, uint32_t parity, uint32_t *err)
{
    for (uint32_t left = 1u << 20; left; left--) {
        if (mbar_try_wait(bar, parity))
            return true;
        __nanosleep(20);
    }
    atomicCAS(err, 0u, (uint32_t)DEV_ERR_MBAR_TIMEOUT);
    return false;
}

// packed f32 pairs
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 c;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(c))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return c;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 c;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(c))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return c;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)),
          "l"(reinterpret_cast<uint64_t &>(c)));
    return d;
}

// A pair that a range begins and does not end.
struct __align__(16) JoinHead {
    int pieces;         // 0: no such pair
    int first, vectors; // of its rows: the first (row, query head) of the KV head, and how many
    int g, r0;          // KV head, first row of the sequence
    int pad[3];
};

// Join the pieces of each pair that no range had to itself.  The tiles of all
// pairs are cut into `slots` consecutive ranges; a range that begins a pair and
// does not end it keeps its piece in its second slot and notes the pair in
// `head`; the ranges behind keep theirs in their first slots.  A piece: the
// unnormalised output [GV][D], then maxima [GV] (in powers of two) and sums
// [GV].  Every block lists the pairs; a task is one vector of one pair.  A warp
// takes a task, or, when there are no more tasks than blocks (one long
// sequence: a hundred pieces and more), the whole block does.  The kernel is a
// chain of a few loads that depend on one another, so each step has all its
// loads in flight at once.
template <class T, int D, int GV>
__global__ void __launch_bounds__(JT) kv8_join_kernel(Kv8Attn a, const float *part, const JoinHead *head, int slots)
{
    constexpr int W = JT / 32, DL = D / 32, PER = (JOIN_SLOTS + JT - 1) / JT;
    constexpr int BATCH = 8; // pieces in flight
    __shared__ int s_owner[JOIN_SLOTS];
    __shared__ int s_n[W];
    __shared__ float s_m[W], s_l[W], s_o[W][D];
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rep = a.n_heads / a.c.n_kv;
    const size_t stride = (size_t)GV * (D + 2);
    int pieces[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; i++)
        pieces[i] = i * JT + (int)threadIdx.x < slots ? head[i * JT + threadIdx.x].pieces : 0;
#pragma unroll
    for (int i = 0; i < PER; i++)
        mine += pieces[i] > 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        upto += lane >= o ? y : 0;
    }
    if (lane == 31)
        s_n[warp] = upto;
    __syncthreads();
    int count = 0, at = upto - mine;
#pragma unroll
    for (int i = 0; i < W; i++) {
        at += i < warp ? s_n[i] : 0;
        count += s_n[i];
    }
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (pieces[i] > 0)
            s_owner[at++] = i * JT + threadIdx.x;
    __syncthreads();
    const bool wide = count * GV <= (int)gridDim.x;
    const int step = wide ? gridDim.x : gridDim.x * W;
    for (int task = wide ? blockIdx.x : blockIdx.x * W + warp; task < count * GV; task += step) {
        const int w = s_owner[task / GV], vi = task % GV;
        const JoinHead h = head[w];
        if (vi >= h.vectors)
            continue; // the same for all of the task's warps
        auto piece = [&](int i) { return part + ((size_t)2 * (w + i) + (i ? 0 : 1)) * stride; };
        const int p0 = wide ? h.pieces * warp / W : 0, p1 = wide ? h.pieces * (warp + 1) / W : h.pieces;
        float m = -INFINITY, l = 0.0f, o[DL], x[BATCH][DL]; // lane i has dims DL * i ..
#pragma unroll
        for (int k = 0; k < DL; k++)
            o[k] = 0.0f;
        for (int i0 = p0; i0 < p1; i0 += 32) {
            const int here = min(32, p1 - i0);
            const float mi = lane < here ? piece(i0 + lane)[(size_t)GV * D + vi] : -INFINITY;
            const float li = lane < here ? piece(i0 + lane)[(size_t)GV * (D + 1) + vi] : 0.0f;
            auto fetch = [&](int b) {
#pragma unroll
                for (int i = 0; i < BATCH; i++) {
                    const float *src = piece(i0 + min(b + i, here - 1)) + (size_t)vi * D + lane * DL;
                    if constexpr (DL == 4) {
                        const float4 y = *reinterpret_cast<const float4 *>(src);
                        x[i][0] = y.x, x[i][1] = y.y, x[i][2] = y.z, x[i][3] = y.w;
                    } else {
                        const float2 y = *reinterpret_cast<const float2 *>(src);
                        x[i][0] = y.x, x[i][1] = y.y;
                    }
                }
            };
            fetch(0);
            const float mn = fmaxf(m, warp_max(mi)), ref = mn == -INFINITY ? 0.0f : mn;
            const float c = ex2(m - ref), e = ex2(mi - ref); // 0 for the lanes behind the last piece
            l = l * c + warp_sum(li * e);
            m = mn;
#pragma unroll
            for (int k = 0; k < DL; k++)
                o[k] *= c;
            for (int b = 0; b < here; b += BATCH) {
                if (b)
                    fetch(b);
#pragma unroll
                for (int i = 0; i < BATCH; i++) {
                    const float ei = __shfl_sync(0xffffffffu, e, (b + i) & 31);
#pragma unroll
                    for (int k = 0; k < DL; k++)
                        o[k] += ei * x[i][k];
                }
            }
        }
        const int v = h.first + vi;
        T *out = reinterpret_cast<T *>(a.out) + (size_t)(h.r0 + v / rep) * a.ld_out + (size_t)(h.g * rep + v % rep) * D;
        if (!wide) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int k = 0; k < DL; k++)
                out[lane * DL + k] = T(o[k] * inv);
            continue;
        }
        __syncthreads(); // the last task's sums are read
#pragma unroll
        for (int k = 0; k < DL; k++)
            s_o[warp][lane * DL + k] = o[k];
        if (lane == 0) {
            s_m[warp] = m;
            s_l[warp] = l;
        }
        __syncthreads();
        if (threadIdx.x < D) {
            float mm = -INFINITY, ll = 0.0f, oo = 0.0f;
#pragma unroll
            for (int i = 0; i < W; i++)
                mm = fmaxf(mm, s_m[i]);
            mm = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int i = 0; i < W; i++) {
                const float e = ex2(s_m[i] - mm);
                ll += s_l[i] * e;
                oo += s_o[i][threadIdx.x] * e;
            }
            out[threadIdx.x] = T(ll == 0.0f ? 0.0f : oo / ll);
        }
    }
}

} // namespace

} // namespace llmrs
