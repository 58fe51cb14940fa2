// kv8_cache.cu - writing and reading the paged 8-bit KV cache (sm_100a).
//
// Append, for each page p and KV head that new rows fall into (x: the new
// rows' values there, keys rotated by their positions first):
//   s1   = max(s0, max|x| / 127)      s0 = 0 when the page held none of the
//                                     sequence's tokens before; s1 < 2^-126 -> 0
//   new  = rint(x * (1 / s1))         older codes c of the page, when s1 > s0:
//                                     rint(c * (s0 / s1))
// Every operation is one f32 rounding (no FMA), so the codes do not depend on
// how the work is split.  No counterpart in the reference: its cache is f32
// and contiguous (src/core/layer.rs:114-128, 219-246).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>

#include "kv8.cuh"

namespace llmrs {

namespace {

constexpr int AP_THREADS = 256;
constexpr int FULL_WARPS = 4; // to a unit of full pages

__device__ __forceinline__ float rot_lo(float lo, float hi, float c, float s)
{
    return __fsub_rn(__fmul_rn(lo, c), __fmul_rn(hi, s));
}
__device__ __forceinline__ float rot_hi(float lo, float hi, float c, float s)
{
    return __fadd_rn(__fmul_rn(lo, s), __fmul_rn(hi, c));
}

// a value that is no number, or infinite, is stored as zero and reported
__device__ __forceinline__ float finite_or_zero(float x, bool &bad)
{
    if (fabsf(x) <= FLT_MAX)
        return x;
    bad = true;
    return 0.0f;
}

// Four codes rint(x * inv).  1.5 * 2^23 added rounds to an integer, to even on a
// tie like rint, and leaves it in the low byte.  No clamp: a new |x| is at most
// 127 s1 (1 + 2^-24) and inv rounds once more, so x * inv stays below 127.0001;
// an old code is multiplied by less than one.
__device__ __forceinline__ uint32_t code4(float4 x, float inv)
{
    auto code = [&](float v) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f)); };
    const uint32_t a = __byte_perm(code(x.x), code(x.y), 0x0040), c = __byte_perm(code(x.z), code(x.w), 0x0040);
    return __byte_perm(a, c, 0x5410);
}

// WARPS warps per (touched page, KV head, K or V), the others of the CTA take
// further heads of the page.  Up to HOLD rows of a thread are loaded at once and
// stay in registers between the maximum and the codes; longer ones are read again,
// from the L2.  Full pages are bound by reading the rows: 8192 rows of 8 heads of
// 128, f32, pages of 32 take 26 us (84 MB: half of the memory's rate, whatever the
// warps, rows held and CTAs per SM).  A few rows per page are a chain of loads
// that depend on one another, so a warp to a unit keeps more of such a batch's
// chains on the GPU at once, and four warps shorten each (append_one_warp).
template <class T, int D, int WARPS>
__global__ void __launch_bounds__(AP_THREADS) kv8_append_kernel(Kv8 c, Kv8Batch b, const T *k, const T *v,
                                                                long long ld, Kv8Rope rope, uint32_t *err)
{
    constexpr int TPR = D / 8;              // threads per row: dims 4j.. and D/2 + 4j..
    constexpr int THREADS = 32 * WARPS;     // of a unit
    constexpr int RPI = THREADS / TPR;      // rows per round
    constexpr int HOLD = 2;
    __shared__ float s_max[AP_THREADS / 32];
    const int page = c.page, unit = blockIdx.y * (AP_THREADS / THREADS) + (int)threadIdx.x / THREADS;
    const int g = unit >> 1, tid = threadIdx.x % THREADS;
    const bool is_v = unit & 1;
    long long within = 0;
    const int s = kv8_find_unit<AP_THREADS>(
        b.n_seqs, blockIdx.x,
        [&](int i) -> long long {
            int r0, n, len;
            kv8_seq(b, i, err, r0, n, len);
            return n ? (len + n - 1) / page - len / page + 1 : 0;
        },
        within);
    if (s < 0 || g >= c.n_kv)
        return;
    int r0, n, len;
    kv8_seq(b, s, err, r0, n, len);
    const int p = len / page + (int)within;
    const int id = kv8_page(b, c, s, p, err);
    if (id < 0)
        return;
    const int t0 = max(len, p * page), t1 = min(len + n, (p + 1) * page); // new positions in this page
    const int held = t0 - p * page;                                      // older tokens in front of them
    const T *src = (is_v ? v : k) + (size_t)(r0 + t0 - len) * ld + (size_t)g * D;
    const size_t at = ((size_t)id * c.n_kv + g);
    int8_t *codes = (is_v ? c.vq : c.kq) + at * page * D;
    float *scale = (is_v ? c.vs : c.ks) + at;
    const float s0 = held ? *scale : 0.0f;
    const int j = tid % TPR, rr = tid / TPR, rows = t1 - t0;
    const bool turn = !is_v && rope.cos;
    bool bad = false;
    bool clean = false; // some value is not finite, and goes as zero
    auto row = [&](int i, float4 &lo, float4 &hi) { // new row i: 4 values of each half, rotated
        const T *x = src + (size_t)i * ld;
        lo = kv8_load4(x + 4 * j);
        hi = kv8_load4(x + D / 2 + 4 * j);
        if (turn) {
            const size_t o = (size_t)(t0 + i) * (D / 2) + 4 * j;
            const float4 cs = *reinterpret_cast<const float4 *>(rope.cos + o);
            const float4 sn = *reinterpret_cast<const float4 *>(rope.sin + o);
            const float4 a = lo, h = hi;
            lo = make_float4(rot_lo(a.x, h.x, cs.x, sn.x), rot_lo(a.y, h.y, cs.y, sn.y),
                             rot_lo(a.z, h.z, cs.z, sn.z), rot_lo(a.w, h.w, cs.w, sn.w));
            hi = make_float4(rot_hi(a.x, h.x, cs.x, sn.x), rot_hi(a.y, h.y, cs.y, sn.y),
                             rot_hi(a.z, h.z, cs.z, sn.z), rot_hi(a.w, h.w, cs.w, sn.w));
        }
        if (clean) {
            lo = make_float4(finite_or_zero(lo.x, bad), finite_or_zero(lo.y, bad), finite_or_zero(lo.z, bad),
                             finite_or_zero(lo.w, bad));
            hi = make_float4(finite_or_zero(hi.x, bad), finite_or_zero(hi.y, bad), finite_or_zero(hi.z, bad),
                             finite_or_zero(hi.w, bad));
        }
    };
    float4 lo[HOLD], hi[HOLD];
    auto largest = [&]() { // of the unit's rows, infinite when a value is not finite
        float m = 0.0f, nan = 0.0f; // a product with zero is zero but for those
        auto see = [&](float x) {
            m = fmaxf(m, fabsf(x));
            nan = fmaf(x, 0.0f, nan);
        };
        for (int i0 = rr; i0 < rows; i0 += HOLD * RPI) {
#pragma unroll
            for (int u = 0; u < HOLD; u++) {
                lo[u] = hi[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (i0 + u * RPI < rows)
                    row(i0 + u * RPI, lo[u], hi[u]);
            }
#pragma unroll
            for (int u = 0; u < HOLD; u++) {
                see(lo[u].x), see(lo[u].y), see(lo[u].z), see(lo[u].w);
                see(hi[u].x), see(hi[u].y), see(hi[u].z), see(hi[u].w);
            }
        }
        m = warp_max(nan == 0.0f ? m : INFINITY);
        if constexpr (WARPS > 1) {
            const int first = (int)threadIdx.x / THREADS * WARPS;
            auto sync = [&]() { // the unit's warps
                asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / THREADS), "n"(THREADS) : "memory");
            };
            sync(); // an earlier call's maxima are read
            if ((threadIdx.x & 31) == 0)
                s_max[threadIdx.x >> 5] = m;
            sync();
#pragma unroll
            for (int w = 0; w < WARPS; w++)
                m = fmaxf(m, s_max[first + w]);
        }
        return m;
    };
    float m = largest();
    if (m == INFINITY) { // the same in the whole unit
        clean = true;
        m = largest();
    }
    float s1 = fmaxf(s0, __fdiv_rn(m, 127.0f));
    if (s1 < FLT_MIN)
        s1 = 0.0f;
    const float inv = s1 > 0.0f ? __fdiv_rn(1.0f, s1) : 0.0f;
    const bool again = rows > HOLD * RPI; // more rows than the registers held
    for (int i0 = rr; i0 < rows; i0 += HOLD * RPI) {
#pragma unroll
        for (int u = 0; u < HOLD; u++) {
            const int i = i0 + u * RPI;
            if (i >= rows)
                continue;
            if (again)
                row(i, lo[u], hi[u]);
            int8_t *dst = codes + (size_t)(held + i) * D;
            *reinterpret_cast<uint32_t *>(dst + 4 * j) = code4(lo[u], inv);
            *reinterpret_cast<uint32_t *>(dst + D / 2 + 4 * j) = code4(hi[u], inv);
        }
    }
    if (s1 > s0 && held) {
        const float ratio = __fdiv_rn(s0, s1);
        for (int w = tid; w < held * D / 16; w += THREADS) {
            int4 x = reinterpret_cast<const int4 *>(codes)[w];
            char4 o[4];
            memcpy(o, &x, 16);
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; e++)
                y[e] = code4(make_float4(o[e].x, o[e].y, o[e].z, o[e].w), ratio);
            reinterpret_cast<uint4 *>(codes)[w] = make_uint4(y[0], y[1], y[2], y[3]);
        }
    }
    if (tid == 0)
        *scale = s1;
    if (bad)
        atomicCAS(err, 0u, (uint32_t)DEV_ERR_NONFINITE);
}

__device__ __forceinline__ void store1(float *p, float x) { *p = x; }
__device__ __forceinline__ void store1(__half *p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void store1(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

// pages back as values: one CTA per (page, KV head, K or V), 16 codes a thread
template <class T>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8 c, const int *pages, T *k, T *v, uint32_t *err)
{
    const int id = pages[blockIdx.x], g = blockIdx.y;
    if (id < 0 || id >= c.n_pages) {
        if (threadIdx.x == 0)
            atomicCAS(err, 0u, (uint32_t)DEV_ERR_BAD_PAGE);
        return;
    }
    const size_t at = (size_t)id * c.n_kv + g, n = (size_t)c.page * c.D;
    const int8_t *codes = (blockIdx.z ? c.vq : c.kq) + at * n;
    const float s = (blockIdx.z ? c.vs : c.ks)[at];
    T *out = (blockIdx.z ? v : k) + ((size_t)blockIdx.x * c.n_kv + g) * n;
    for (size_t i = (size_t)threadIdx.x * 16; i < n; i += 256 * 16) {
        const int4 w = *reinterpret_cast<const int4 *>(codes + i);
        int8_t q[16];
        memcpy(q, &w, 16);
        __align__(16) T o[16];
#pragma unroll
        for (int e = 0; e < 16; e++)
            store1(&o[e], __fmul_rn((float)q[e], s));
#pragma unroll
        for (int e = 0; e < (int)sizeof(T); e++)
            reinterpret_cast<int4 *>(out + i)[e] = reinterpret_cast<const int4 *>(o)[e];
    }
}

// Whether a warp takes a unit, in place of four: yes for a row or two per sequence, and up to
// 32 while the units are many for the rows.  Both forms, us, f32 rows, 8 KV heads of 128, pages
// of 64, one warp / four:
//   sequences   1 row      3 rows     6 rows     9 rows     16 rows     32 rows     64 rows
//     8         3.2/3.2    3.5/3.3    4.2/3.3    5.2/3.5     6.5/3.6    10.8/5.0
//    32                               4.4/4.4    5.3/4.8     7.3/5.0
//    64         3.4/4.2    3.9/6.2    4.8/6.6    5.8/7.1     7.7/7.4    13.0/10.6
//   191         4.3/9.5    5.5/13.4   6.7/14.2   8.0/15.3   11.2/16.6   20.0/24.4   52.4/44.9
// They cross at rows = units / 64 to units / 85, units = 2 x KV heads x sequences (so also for 2
// KV heads), and for heads of 64, twice as many to a warp's round, at twice that.  Where the
// scale grows, one warp takes 7 us longer for a page of 103 held tokens, four take 2.
bool append_one_warp(const Kv8 &c, const Kv8Batch &b)
{
    const long long rows = (b.n_rows + (long long)b.n_seqs - 1) / b.n_seqs; // of a sequence, on average
    const long long units = 2LL * c.n_kv * b.n_seqs;
    return rows <= 2 || (rows <= 32 && rows * c.D * 80 <= units * 128);
}

template <class T, int D>
cudaError_t append_d(const Kv8 &c, const Kv8Batch &b, const T *k, const T *v, long long ld, const Kv8Rope &r,
                     uint32_t *err, unsigned pages, cudaStream_t stream)
{
    auto run = [&](auto kernel, int warps) {
        const int per = AP_THREADS / 32 / warps; // units of a CTA
        return launch(kernel, dim3(pages, (2 * c.n_kv + per - 1) / per), dim3(AP_THREADS), 0, stream, false, c, b, k, v, ld,
                      r, err);
    };
    if (append_one_warp(c, b))
        return run(kv8_append_kernel<T, D, 1>, 1);
    return run(kv8_append_kernel<T, D, FULL_WARPS>, FULL_WARPS);
}

template <class T>
cudaError_t append_t(const Kv8 &c, const Kv8Batch &b, const void *k, const void *v, long long ld, const Kv8Rope &r,
                     uint32_t *err, unsigned pages, cudaStream_t stream)
{
    const T *kt = reinterpret_cast<const T *>(k), *vt = reinterpret_cast<const T *>(v);
    if (c.D == 128)
        return append_d<T, 128>(c, b, kt, vt, ld, r, err, pages, stream);
    return append_d<T, 64>(c, b, kt, vt, ld, r, err, pages, stream);
}

} // namespace

int kv8_append(const Kv8 &c, const Kv8Batch &b, const void *k, const void *v, int dtype, long long ld,
               const Kv8Rope &r, uint32_t *err, cudaStream_t stream)
{
    // n rows of one sequence touch at most n pages, and at most n/page + 2
    const long long units = std::min((long long)b.n_rows, (long long)b.n_rows / c.page + 2LL * b.n_seqs);
    const unsigned grid = (unsigned)units;
    if (dtype == LLMRS_F32)
        LLMRS_CUDA_TRY(append_t<float>(c, b, k, v, ld, r, err, grid, stream));
    else if (dtype == LLMRS_BF16)
        LLMRS_CUDA_TRY(append_t<__nv_bfloat16>(c, b, k, v, ld, r, err, grid, stream));
    else
        LLMRS_CUDA_TRY(append_t<__half>(c, b, k, v, ld, r, err, grid, stream));
    return LLMRS_OK;
}

int kv8_read(const Kv8 &c, const int *pages, int n, void *k, void *v, int dtype, uint32_t *err, cudaStream_t stream)
{
    const dim3 grid((unsigned)n, (unsigned)c.n_kv, 2), block(256);
    if (dtype == LLMRS_F32)
        LLMRS_CUDA_TRY(launch(kv8_read_kernel<float>, grid, block, 0, stream, false, c, pages, (float *)k, (float *)v,
                              err));
    else if (dtype == LLMRS_BF16)
        LLMRS_CUDA_TRY(launch(kv8_read_kernel<__nv_bfloat16>, grid, block, 0, stream, false, c, pages,
                              (__nv_bfloat16 *)k, (__nv_bfloat16 *)v, err));
    else
        LLMRS_CUDA_TRY(launch(kv8_read_kernel<__half>, grid, block, 0, stream, false, c, pages, (__half *)k,
                              (__half *)v, err));
    return LLMRS_OK;
}

} // namespace llmrs
