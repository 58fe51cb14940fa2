// verify.cu - verification of drafted tokens against the target's
// probabilities, from given uniform draws (sm_100a).
//
// A sequence with k drafts d_0 .. d_{k-1} has k + 1 rows of target logits; row
// i gives p_i = softmax(logits_i / temperature), and q_i is the distribution
// that d_i was drawn from.
//   accept d_i while u_i * q_i(d_i) < p_i(d_i)      (probability min(1, p/q))
//   at the first rejection, i = a: the next token comes from max(p_a - q_a, 0),
//   after k acceptances from p_k, by the inverse CDF in index order: the first
//   token whose running sum exceeds u_k * total.
// The tokens that come out are distributed as if drawn from p row by row.
// Temperature 0 makes p one at the row's first maximum.  The reference draws
// one token at a time on the host (src/main.rs:192-305).
//
// Two kernels.  verify_rows: every row's maximum and sum of exponentials, one
// CTA per (row, chunk of VCHUNK tokens), all of a thread's 16-byte loads in
// flight at once; bound by reading the logits once (35 us for 148 MB, 288 rows
// of 128256 f32 logits).  verify_pick: a cluster of CTAs per sequence decides
// the acceptances, then takes the one row that the next token comes from twice,
// for its sum and for what is left of it, each warp a range of consecutive
// tokens; the CTA whose warp holds the draw looks through that range once more.
// Exponentials and sums are in 64 bits here: a draw next to the border of two
// tokens would otherwise be decided by the rounding of a 32-bit running sum
// over the whole vocabulary.  (An acceptance is one comparison with p of one
// token, whose sum of f32 exponentials, 32 at a time in f32 and then in 64 bits,
// leaves p off by less than 2^-18 of itself: an exponential by 2^-22, 32 of them
// added by 2^-19.)  54 us for 64 such sequences, of which 4 for the
// acceptances, 20 and 27 for the two passes (half of it conversions and 64-bit
// arithmetic) and 2 for the end; a warp alone in its range's last look took 40.
// (64-bit exponentials of every row in verify_rows save the first pass here
// and cost more: 31 us.)
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>
#include <limits.h>
#include <math.h>

#include "common.cuh"
#include "verify.cuh"

namespace cg = cooperative_groups;

namespace llmrs {

namespace {

constexpr int VT = 256;         // threads of verify_rows
constexpr int VPER = 32;        // logits a thread holds
constexpr int VCHUNK = VT * VPER;
constexpr int PT = 512;         // threads of verify_pick
constexpr int PW = PT / 32;
constexpr int PPER = 16;        // tokens of a thread in flight

// a chunk's part of its row's statistics
struct RowPart {
    float m;      // maximum
    int at;       // its first place
    double s;     // sum of exp((l - m) / T)
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// a logit that is no number has no weight; infinite ones share it
__device__ __forceinline__ float clean(float l)
{
    return l != l ? -INFINITY : fminf(l, FLT_MAX);
}

__device__ __forceinline__ double warp_sum_d(double v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// largest value, the lower place on a tie
__device__ __forceinline__ void warp_best(float &m, int &at)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o);
        const int a2 = __shfl_xor_sync(0xffffffffu, at, o);
        if (m2 > m || (m2 == m && a2 < at)) {
            m = m2;
            at = a2;
        }
    }
}

// exp(x) for x <= 0, whole warp, by argument reduction to a table of powers and
// the Taylor polynomial (the table-driven method of P. T. P. Tang, ACM TOMS 15,
// 1989); table: 2^(lane / 32).  x = n ln2/32 + r with |r| <= ln2/64, exp(x) =
// 2^(n/32) (1 + r + r^2/2 + r^3/6 + r^4/24), off by r^5/120 < 1.25e-12 of itself
// (n times the rounding of ln2/32 adds 4e-14 at the most); exact for x = 0; below
// -700 (and for NaN) 0.
__device__ __forceinline__ double exp64(double x, double table)
{
    const bool some = x > -700.0;
    x = some ? x : 0.0;
    const int n = __double2int_rn(x * 46.166241308446828384);
    const double r = fma((double)n, -0.021660849392498290195, x);
    const double y = fma(fma(fma(fma(r, 1.0 / 24, 1.0 / 6), r, 0.5), r, 1.0), r, 1.0) * __shfl_sync(0xffffffffu, table, n & 31);
    return some ? __hiloint2double(__double2hiint(y) + ((n >> 5) << 20), __double2loint(y)) : 0.0;
}

template <class T>
__global__ void __launch_bounds__(VT) verify_rows_kernel(VerifyParams p, RowPart *part, int n_chunks)
{
    __shared__ float s_m[VT / 32];
    __shared__ int s_at[VT / 32];
    __shared__ double s_s[VT / 32];
    __shared__ int s_seq;
    constexpr int E = 16 / (int)sizeof(T); // logits of a 16-byte load
    const int row = blockIdx.y, chunk = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T *x = reinterpret_cast<const T *>(p.logits) + (size_t)row * p.ld;
    griddep_launch_dependents();
    // loads on 16-byte boundaries whatever the row's: load v of the row covers the tokens E*v - skew ..
    const int skew = (int)(((uintptr_t)x & 15) / sizeof(T)), c0 = chunk * VCHUNK - skew;
    float l[VPER];
#pragma unroll
    for (int i = 0; i < VPER / E; i++) {
        const int t = c0 + (i * VT + (int)threadIdx.x) * E;
        if (t >= 0 && t + E <= p.vocab) {
            const uint4 w = __ldcs(reinterpret_cast<const uint4 *>(x + t));
            T v[E];
            memcpy(v, &w, 16);
#pragma unroll
            for (int e = 0; e < E; e++)
                l[i * E + e] = to_float(v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < E; e++)
                l[i * E + e] = t + e >= 0 && t + e < p.vocab ? to_float(x[t + e]) : -INFINITY;
        }
    }
    // the row's sequence, for its temperature: the first that holds it (row starts that fall
    // end the batch for verify_pick, and in front of them no other sequence does)
    float T_ = 1.0f;
    if (p.temperature) {
        if (threadIdx.x == 0)
            s_seq = INT_MAX;
        __syncthreads();
        for (int s = threadIdx.x; s < p.n_seqs; s += VT)
            if (p.row_start[s] <= row && row < p.row_start[s + 1])
                atomicMin(&s_seq, s);
        __syncthreads();
        if (s_seq != INT_MAX)
            T_ = p.temperature[s_seq];
    }
    // a subnormal temperature's reciprocal is past f32: it and the differences of the logits
    // take 2^64 each (a difference that this makes infinite weighs nothing either way)
    const bool tiny = T_ > 0.0f && T_ < FLT_MIN;
    const float inv = T_ > 0.0f ? 1.4426950408889634f / (tiny ? T_ * 0x1p64f : T_) : 0.0f;
    float m = -INFINITY;
    int at = INT_MAX;
#pragma unroll
    for (int i = 0; i < VPER; i++) {
        l[i] = clean(l[i]);
        if (l[i] > m) {
            m = l[i];
            at = c0 + ((i / E) * VT + (int)threadIdx.x) * E + i % E;
        }
    }
    warp_best(m, at);
    if (lane == 0) {
        s_m[warp] = m;
        s_at[warp] = at;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < VT / 32; w++)
        if (s_m[w] > m || (s_m[w] == m && s_at[w] < at)) {
            m = s_m[w];
            at = s_at[w];
        }
    float sum = 0.0f;
    if (tiny) {
#pragma unroll
        for (int i = 0; i < VPER; i++)
            sum += l[i] > -INFINITY ? ex2((l[i] - m) * 0x1p64f * inv) : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < VPER; i++)
            sum += l[i] > -INFINITY ? ex2((l[i] - m) * inv) : 0.0f;
    }
    const double d = warp_sum_d((double)sum);
    if (lane == 0)
        s_s[warp] = d;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int w = 0; w < VT / 32; w++)
            s += s_s[w];
        RowPart r;
        r.m = m;
        r.at = at;
        r.s = s;
        part[(size_t)row * n_chunks + chunk] = r;
    }
}

// a row's statistics from its chunks (whole warp)
__device__ __forceinline__ RowPart row_stats(const RowPart *part, int n_chunks, double inv)
{
    const int lane = threadIdx.x & 31;
    RowPart r;
    r.m = -INFINITY;
    r.at = INT_MAX;
    for (int c = lane; c < n_chunks; c += 32)
        if (part[c].m > r.m) {
            r.m = part[c].m;
            r.at = part[c].at;
        }
    warp_best(r.m, r.at);
    double s = 0.0;
    for (int c = lane; c < n_chunks; c += 32)
        if (part[c].m > -INFINITY)
            s += part[c].s * exp(((double)part[c].m - (double)r.m) * inv);
    r.s = warp_sum_d(s);
    return r;
}

// Four logits of a row from token t on, -inf outside of [0, vocab); t lies on a
// boundary of four elements of the row's memory.
template <class T>
__device__ __forceinline__ void load4(const T *x, int t, int vocab, float (&v)[4])
{
    if (t >= 0 && t + 4 <= vocab) {
        T w[4];
        if constexpr (sizeof(T) == 4) {
            const uint4 raw = *reinterpret_cast<const uint4 *>(x + t);
            memcpy(w, &raw, 16);
        } else {
            const uint2 raw = *reinterpret_cast<const uint2 *>(x + t);
            memcpy(w, &raw, 8);
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            v[e] = clean(to_float(w[e]));
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            v[e] = t + e >= 0 && t + e < vocab ? clean(to_float(x[t + e])) : -INFINITY;
    }
}

// the same tokens of a row of draft probabilities, of any alignment; 0 outside
__device__ __forceinline__ void load_q4(const float *q, int t, int vocab, bool wide, float (&v)[4])
{
    if (wide && t >= 0 && t + 4 <= vocab) {
        const float4 w = __ldcs(reinterpret_cast<const float4 *>(q + t));
        v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            v[e] = t + e >= 0 && t + e < vocab ? q[t + e] : 0.0f;
    }
}

// the sum over the CTA, in every thread; s_red: PW + 1 places, free at entry
__device__ __forceinline__ double cta_sum(double v, double *s_red)
{
    const int lane = threadIdx.x & 31;
    v = warp_sum_d(v);
    if (lane == 0)
        s_red[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum_d(lane < PW ? s_red[lane] : 0.0);
}

template <class T, int PICK_CTAS>
__global__ void __launch_bounds__(PT, 2) verify_pick_kernel(VerifyParams p, const RowPart *part, int n_chunks)
{
    constexpr int PWARPS = PICK_CTAS * PW;
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ int s_first;                   // first rejected draft
    __shared__ double s_red[PW];
    __shared__ double s_z[PICK_CTAS];         // each CTA's share of the row's sum
    __shared__ double s_w[2][PWARPS];         // each warp's share: of max(p - q, 0), of p
    __shared__ int s_final[2][PWARPS];        // last token with weight in each warp's range
    __shared__ int s_hit;
    griddep_wait();
    const int seq = blockIdx.x / PICK_CTAS, rank = (int)cluster.block_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r0 = p.row_start[seq], r1 = p.row_start[seq + 1], n = r1 - r0;
    if (n <= 0 || r0 < 0 || r1 > p.n_rows) { // the same for the whole cluster
        if (rank == 0 && threadIdx.x == 0) {
            p.accepted[seq] = 0;
            if (n != 0)
                atomicCAS(p.err, 0u, (uint32_t)DEV_ERR_BAD_BATCH);
        }
        return;
    }
    // drafts lie packed without the last rows: one less than the rows for each
    // sequence in front that has any
    int in_front = 0;
    bool rising = p.row_start[0] >= 0;
    for (int i0 = 0; i0 < seq; i0 += PT) {
        const int i = i0 + (int)threadIdx.x, rows = i < seq ? p.row_start[i + 1] - p.row_start[i] : 0;
        in_front += __syncthreads_count(rows > 0);
        rising = !__syncthreads_or(rows < 0) && rising;
    }
    const int k = n - 1, d0 = r0 - p.row_start[0] - in_front; // drafts and their first place
    if (!rising || (k > 0 && d0 + k > p.n_drafts)) { // or more drafts than there are
        if (rank == 0 && threadIdx.x == 0) {
            p.accepted[seq] = 0;
            atomicCAS(p.err, 0u, (uint32_t)DEV_ERR_BAD_BATCH);
        }
        return;
    }
    const float T_ = p.temperature ? p.temperature[seq] : 1.0f;
    const bool greedy = !(T_ > 0.0f);
    const double inv = greedy ? 1.0 : 1.0 / (double)T_;
    if (threadIdx.x == 0)
        s_first = k;
    __syncthreads();
    for (int i = warp; i < k; i += PW) {
        const int row = r0 + i, d = p.draft[d0 + i];
        const RowPart r = row_stats(part + (size_t)row * n_chunks, n_chunks, inv);
        if (lane == 0) {
            double pd = 0.0;
            if (d < 0 || d >= p.vocab)
                atomicCAS(p.err, 0u, (uint32_t)DEV_ERR_BAD_TOKEN);
            else if (greedy)
                pd = d == r.at ? 1.0 : 0.0;
            else if (r.m > -INFINITY) {
                const float l = clean(to_float(reinterpret_cast<const T *>(p.logits)[(size_t)row * p.ld + d]));
                pd = exp(((double)l - (double)r.m) * inv) / r.s;
            }
            const bool known = d >= 0 && d < p.vocab;
            const double qd = p.q && known ? (double)p.q[(size_t)(d0 + i) * p.ldq + d] : 1.0;
            if (!((double)p.u[row] * qd < pd))
                atomicMin(&s_first, i);
            if (rank == 0 && p.probs)
                p.probs[row] = (float)pd; // overwritten below behind the first rejection
        }
    }
    __syncthreads();
    const int a = s_first, row = r0 + a;
    if (rank == 0)
        for (int i = threadIdx.x; i < n; i += PT) {
            if (i != a)
                p.tokens[r0 + i] = i < a ? p.draft[d0 + i] : -1;
            if (i > a && p.probs)
                p.probs[r0 + i] = 0.0f;
            if (i == 0)
                p.accepted[seq] = a;
        }
    const RowPart r = row_stats(part + (size_t)row * n_chunks, n_chunks, inv);
    if (greedy || !(r.m > -INFINITY)) { // the first maximum; no token when every one is masked
        if (rank == 0 && threadIdx.x == 0) {
            const bool some = r.m > -INFINITY;
            p.tokens[row] = some ? r.at : -1;
            if (p.probs)
                p.probs[row] = some ? 1.0f : 0.0f;
        }
        return;
    }
    cluster.barrier_arrive(); // every CTA has begun before another writes to its shared memory
    const T *x = reinterpret_cast<const T *>(p.logits) + (size_t)row * p.ld;
    const bool rest = a < k;
    const float *q = rest && p.q ? p.q + (size_t)(d0 + a) * p.ldq : nullptr;
    const int gone = rest && !p.q ? p.draft[d0 + a] : -1; // a certain draft's own token
    // warp `gw` of the cluster's warps owns the tokens [t0, t1); the ranges' ends lie on
    // boundaries of four elements in memory, the row's own ends mask the rest
    const int skew = (int)(((uintptr_t)x / sizeof(T)) & 3), gw = rank * PW + warp;
    const int per = ((p.vocab + skew + 3) / 4 + PWARPS - 1) / PWARPS * 4;
    const int t0 = min(p.vocab, gw * per - skew), t1 = min(p.vocab, (gw + 1) * per - skew);
    const bool wide = q && ((uintptr_t)(q - skew) & 15) == 0;
    const double table = exp2((double)lane / 32);
    auto weight = [&](float l) { return exp64(((double)l - (double)r.m) * inv, table); };
    double z = 0.0;
    for (int b = t0; b < t1; b += 32 * PPER) {
        float v[PPER / 4][4];
#pragma unroll
        for (int k = 0; k < PPER / 4; k++)
            load4(x, b + (k * 32 + lane) * 4, t1, v[k]);
#pragma unroll
        for (int k = 0; k < PPER; k++)
            z += weight(v[k / 4][k % 4]);
    }
    z = cta_sum(z, s_red);
    cluster.barrier_wait();
    if (threadIdx.x < PICK_CTAS)
        cluster.map_shared_rank(s_z, threadIdx.x)[rank] = z;
    cluster.sync();
    z = 0.0;
    for (int c = 0; c < PICK_CTAS; c++)
        z += s_z[c];
    const double invz = 1.0 / z;
    // what is left of token t: max(p - q, 0), without a certain draft's own token
    auto residual = [&](int t, double pt, float qt) {
        const double w = t == gone ? 0.0 : pt - (double)qt;
        return w > 0.0 ? w : 0.0;
    };
    double sw = 0.0, sp = 0.0;
    int fw = -1, fp = -1;
    for (int b = t0; b < t1; b += 32 * PPER) {
        float v[PPER / 4][4], qt[PPER / 4][4] = {};
#pragma unroll
        for (int k = 0; k < PPER / 4; k++) {
            const int t = b + (k * 32 + lane) * 4;
            load4(x, t, t1, v[k]);
            if (q)
                load_q4(q, t, t1, wide, qt[k]);
        }
#pragma unroll
        for (int k = 0; k < PPER; k++) {
            const int t = b + (k / 4 * 32 + lane) * 4 + k % 4;
            const double pt = weight(v[k / 4][k % 4]) * invz, w = residual(t, pt, qt[k / 4][k % 4]);
            sw += w;
            sp += pt;
            fw = w > 0.0 ? t : fw;
            fp = pt > 0.0 ? t : fp;
        }
    }
    sw = warp_sum_d(sw);
    sp = warp_sum_d(sp);
    fw = __reduce_max_sync(0xffffffffu, fw);
    fp = __reduce_max_sync(0xffffffffu, fp);
    if (lane < PICK_CTAS) {
        cluster.map_shared_rank(&s_w[0][0], lane)[gw] = sw;
        cluster.map_shared_rank(&s_w[1][0], lane)[gw] = sp;
        cluster.map_shared_rank(&s_final[0][0], lane)[gw] = fw;
        cluster.map_shared_rank(&s_final[1][0], lane)[gw] = fp;
    }
    cluster.sync(); // the last access to another CTA's shared memory
    // the warp whose range the draw falls into: lane i looks at warps WL * i ..
    constexpr int WL = PWARPS / 32;
    double own[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < WL; i++) {
        own[0] += s_w[0][lane * WL + i];
        own[1] += s_w[1][lane * WL + i];
    }
    const int use = warp_sum_d(own[0]) > 0.0 ? 0 : 1; // p equals q: nothing is left over, draw from p
    auto scan = [&](double c) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o)
                c += y;
        }
        return c;
    };
    double before = scan(use ? own[1] : own[0]);
    const double target = (double)p.u[r1 - 1] * __shfl_sync(0xffffffffu, before, 31);
    before -= use ? own[1] : own[0];
    int owner = -1, last = -1;
    double until = 0.0; // the sum in front of the owner
#pragma unroll
    for (int i = 0; i < WL; i++) {
        const int w = lane * WL + i;
        if (s_final[use][w] >= 0) {
            last = w;
            if (owner < 0 && before + s_w[use][w] > target) {
                owner = w;
                until = before;
            }
        }
        before += s_w[use][w];
    }
    last = __reduce_max_sync(0xffffffffu, last);
    const unsigned found = __ballot_sync(0xffffffffu, owner >= 0);
    const bool past = !found; // the draw lies behind the rounded sum
    const int from = past ? 0 : __ffs(found) - 1;
    owner = past ? last : __shfl_sync(0xffffffffu, owner, from);
    until = __shfl_sync(0xffffffffu, until, from);
    if (owner / PW != rank)
        return;
    // the owner's CTA walks the range, four consecutive tokens of a thread, their sums scanned
    const int o0 = owner * per - skew, o1 = min(p.vocab, o0 + per);
    for (int b = o0; b < o1 && !past; b += PT * 4) {
        const int t = b + (int)threadIdx.x * 4;
        float v[4], qt[4] = {};
        load4(x, t, o1, v);
        if (q)
            load_q4(q, t, o1, wide, qt);
        double pt[4], w[4], mine = 0.0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            pt[e] = weight(v[e]) * invz;
            w[e] = use ? pt[e] : residual(t + e, pt[e], qt[e]);
            mine += w[e];
        }
        const double c = scan(mine);
        __syncthreads();
        if (threadIdx.x == 0)
            s_hit = INT_MAX;
        if (lane == 31)
            s_red[warp] = c;
        __syncthreads();
        const double ends = scan(lane < PW ? s_red[lane] : 0.0); // of the warps
        double front = until + (c - mine) + (warp ? __shfl_sync(0xffffffffu, ends, warp - 1) : 0.0), at = 0.0;
        until += __shfl_sync(0xffffffffu, ends, 31);
        int hit = INT_MAX;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            front += w[e];
            if (hit == INT_MAX && w[e] > 0.0 && front > target) {
                hit = t + e;
                at = pt[e];
            }
        }
        const int first = __reduce_min_sync(0xffffffffu, hit);
        if (lane == 0 && first != INT_MAX)
            atomicMin(&s_hit, first);
        __syncthreads();
        if (s_hit != INT_MAX) {
            if (hit == s_hit) {
                p.tokens[row] = hit;
                if (p.probs)
                    p.probs[row] = (float)at;
            }
            return;
        }
    }
    // no running sum exceeds the target: the last token with weight
    const int token = s_final[use][owner];
    if (threadIdx.x == 0) {
        p.tokens[row] = token;
        if (p.probs)
            p.probs[row] = (float)(exp(((double)clean(to_float(x[token])) - (double)r.m) * inv) * invz);
    }
}

// a row that starts off a 16-byte boundary reaches up to 7 tokens further
int chunks(int vocab) { return (vocab + 7 + VCHUNK - 1) / VCHUNK; }

template <class T, int CTAS>
int pick(const VerifyParams &p, const RowPart *part, int n_chunks, cudaStream_t stream)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.n_seqs * CTAS);
    cfg.blockDim = dim3(PT);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.n_rows > 0 ? 2 : 1;
    LLMRS_CUDA_TRY(cudaLaunchKernelEx(&cfg, verify_pick_kernel<T, CTAS>, p, part, n_chunks));
    return LLMRS_OK;
}

template <class T>
cudaError_t prepare()
{
    return cudaFuncSetAttribute(verify_pick_kernel<T, 16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}

template <class T>
int run(const VerifyParams &p, RowPart *part, cudaStream_t stream)
{
    const int n_chunks = chunks(p.vocab);
    if (p.n_rows > 0)
        LLMRS_CUDA_TRY(launch(verify_rows_kernel<T>, dim3(n_chunks, p.n_rows), dim3(VT), 0, stream, false, p, part,
                              n_chunks));
    // the largest cluster with which all sequences' clusters fit at once, two CTAs an SM
    if (p.n_seqs * 16 <= 296)
        return pick<T, 16>(p, part, n_chunks, stream);
    if (p.n_seqs * 8 <= 296)
        return pick<T, 8>(p, part, n_chunks, stream);
    return pick<T, 4>(p, part, n_chunks, stream);
}

} // namespace

size_t verify_workspace(int n_rows, int vocab)
{
    return (size_t)n_rows * chunks(vocab) * sizeof(RowPart);
}

int verify_prepare(void)
{
    cudaError_t e = prepare<float>();
    if (e == cudaSuccess)
        e = prepare<__half>();
    if (e == cudaSuccess)
        e = prepare<__nv_bfloat16>();
    if (e != cudaSuccess)
        return fail(LLMRS_ECUDA, "verification kernel attributes: %s", cudaGetErrorString(e));
    return LLMRS_OK;
}

int verify_launch(const VerifyParams &p, void *ws, cudaStream_t stream)
{
    RowPart *part = reinterpret_cast<RowPart *>(ws);
    if (p.dtype == LLMRS_F32)
        return run<float>(p, part, stream);
    if (p.dtype == LLMRS_BF16)
        return run<__nv_bfloat16>(p, part, stream);
    return run<__half>(p, part, stream);
}

} // namespace llmrs
