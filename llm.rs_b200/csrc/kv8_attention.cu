// kv8_attention.cu - causal attention of a ragged batch over the paged 8-bit
// KV cache (sm_100a): the kernel for few rows per sequence, its merge, and the
// launch of both paths.
//
// Row i of sequence s stands at position P = lens[s] + i and attends to the
// positions 0 .. P of its pages (its own key and value are in the cache):
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q.k_t - max),
//   k_t = ks * kq_t,  v_t = vs * vq_t,  ks, vs the scales of t's page and head,
// in one pass with the running maximum and sum of the softmax.  q is rotated
// by its position on the way.  The reference's per-head loop
// (src/core/layer.rs:175-333) is the same formula over one sequence's
// contiguous f32 cache.
//
// Few rows: bound by reading the codes once.  The (row, query head) vectors
// that share a KV head are the columns of mma.sync.m16n8k16: S = K Q^T, then
// O^T = V^T P, so a tile of 32 tokens is the long side and few vectors waste
// little.  int8 codes are exact in f16.  f32 rows: q and the probabilities are
// split into two f16 pieces (22 bits and more), the pieces are columns of
// their own in the same instruction, so one pass over the codes serves both.
// f16 rows are split too: with one piece each, the roundings of q and P put
// 3.4e-4 on the result where rounding the result itself costs 2.1e-4.  bf16 rows:
// two pieces of the rotated q, whose errors a sharp head's softmax multiplies, and
// one of P, 11 bits to the result's 8.  q's small pieces are not columns of their own
// but multiplied into the same sums.  One sequence of 131000 tokens, 64 heads over 8,
// 2-norm error and time: 1.64e-3 to 1.69e-3 by the input, the rounding of the result
// alone, and 70 us; with one piece of q 1.69e-3 to 1.83e-3 (scores of some tens: several
// times the rounding) and 65 us; with both of P in columns too as now and 85 us.
//
// Work: the tiles of all (sequence, vector group, KV head) pairs in one row,
// cut into equal ranges, one per warp, whatever the lengths.  A warp streams
// its range through its own ring of shared memory (TMA boxes, swizzled so that
// both fragment patterns read without bank conflicts; K and V of a tile are
// refilled apart) and never waits for another warp.  A pair that lies within one
// range is finished there; the pieces of the others go to the workspace and a
// second kernel joins them in order, so results do not depend on timing.
// Ranges of one CTA side by side, joined in the CTA, shorten the second kernel
// and lengthen this one by more (16 sequences of up to 6 rows: 62 us, then 75):
// short pairs bunch on an SM.
//
// 64 sequences of 37 to 8192 tokens, f32, 32 heads of 128 over 8: 105 us here and 6
// in the join for 542 MB (83 us at the memory's rate).  131000 tokens, bf16, 64 heads
// over 8: 58 and 10 us for 268 MB (41).  A launch without work takes 8 us: finding
// the range, the pages, their scales and q, each a trip to memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "gemv.cuh"
#include "kv8_core.cuh"
#include "kv8_many.cuh"

namespace llmrs {

namespace {

constexpr int FT = 32;        // tokens of a tile
// warps of a CTA by column tiles: as many as the registers of a thread allow
constexpr int few_warps(int nt) { return nt == 1 ? 12 : 8; }
constexpr int F_MAX_CTAS = JOIN_SLOTS / few_warps(1);

struct FewParams {
    CUtensorMap tk, tv; // code pools as rows of D bytes
    Kv8Attn a;
    float *part;        // [warps][2][vectors][D + 2]
    JoinHead *head;     // [warps]
    int many;           // sequences with more vectors per KV head than this are another kernel's
};

// what a warp needs to know of one tile
struct __align__(16) Tile {
    int row0, row1;         // pool rows of its 16-token halves (row1: only for pages of 16); -1: not there
    float ks0, ks1, vs0, vs1;
    int s, pair, tile;      // sequence, its KV head and group, and the tile's index in the pair
    int len, r0, n;         // of the sequence: cached tokens, first row, rows
    __device__ int n_tiles() const { return (int)(((long long)len + n + FT - 1) / FT); }
};
static_assert(sizeof(Tile) == 48, "three 16-byte words");

// whether q's small pieces, where they go into the sums of the large ones, lie in shared
// memory: 16 columns of 128 dims and both pieces do not fit the registers
template <int D, bool SPLIT, int NT>
constexpr bool q_low_shared()
{
    return !SPLIT && NT == 2 && D == 128;
}

template <int D, bool SPLIT, int NT>
struct FewLay {
    static constexpr int FW = few_warps(NT);
    static constexpr bool QLS = q_low_shared<D, SPLIT, NT>();
    static constexpr int STAGES = (NT == 1 || QLS ? 2 : 3) * (128 / D);
    static constexpr int BOX = FT * D;            // bytes of K or V codes of a tile
    static constexpr int RING = STAGES * 2 * BOX; // per warp
    static constexpr int BATCH = 32;              // tile records made at a time
    static constexpr int TILES = BATCH + 16;      // and held per warp
    static constexpr int tile_off = FW * RING;
    static constexpr int ql_off = tile_off + FW * TILES * (int)sizeof(Tile);
    static constexpr int bar_off = ql_off + (QLS ? FW * NT * D * 16 : 0);
    static constexpr int bytes = bar_off + FW * STAGES * 16 + 1024; // + alignment slack
    static_assert(bytes <= 232448 - 1024, "shared memory of one CTA, beside the static part");
};

__device__ __forceinline__ void tma_box(void *dst, const CUtensorMap *map, int row, uint64_t *bar, uint64_t policy)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_addr(dst)),
        "l"(map), "r"(0), "r"(row), "r"(smem_addr(bar)), "l"(policy)
        : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same from nothing
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// (row, head) vectors of one KV head that a CTA's columns hold
template <bool SPLIT, int NT>
constexpr int group_vectors()
{
    return SPLIT ? 4 * NT : 8 * NT;
}

// tiles of all pairs of sequence s
template <int GV>
__device__ __forceinline__ long long seq_tiles(const FewParams &p, int n, int len, int &tiles, int &groups)
{
    const int vectors = n * (p.a.n_heads / p.a.c.n_kv);
    tiles = (int)(((long long)len + n + FT - 1) / FT);
    groups = vectors > p.many ? 0 : (vectors + GV - 1) / GV;
    return (long long)tiles * groups * p.a.c.n_kv;
}

// T: type of the rows; SPLIT: both pieces of q and P are columns of their own, in place of q's
// small pieces being multiplied into the sums of the large ones (bf16 rows); NT: columns / 8
template <class T, int D, bool SPLIT, int NT>
__global__ void __launch_bounds__(few_warps(NT) * 32, 1) kv8_few_kernel(const __grid_constant__ FewParams p)
{
    using Lay = FewLay<D, SPLIT, NT>;
    constexpr int FW = Lay::FW;
    constexpr int GV = group_vectors<SPLIT, NT>();
    constexpr int KS = D / 16;    // k steps of q.k
    constexpr int LD = D / 4;     // dims of q.k a lane holds: LD*t ..
    constexpr int LV = D / 8;     // dims of the output a lane holds: LV*gl ..
    constexpr int MT = D / 16;    // 16-dim tiles of the output
    constexpr int ST = Lay::STAGES;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, t4 = lane & 3;
    const Kv8Attn &a = p.a;
    const int rep = a.n_heads / a.c.n_kv, page = a.c.page;
    griddep_launch_dependents();

    uint8_t *ring = smem + warp * Lay::RING;
    Tile *rec = reinterpret_cast<Tile *>(smem + Lay::tile_off) + warp * Lay::TILES;
    uint64_t *bar = reinterpret_cast<uint64_t *>(smem + Lay::bar_off) + warp * 2 * ST; // K, V of a stage
    if (lane == 0) {
        for (int i = 0; i < 2 * ST; i++)
            mbar_init(&bar[i], 1);
        fence_mbar_init();
    }

    // ---- this warp's range of tiles: warp `slot` of all warps, numbered so that
    // few tiles spread over all SMs
    __shared__ long long s_sum[FW], s_at[FW];
    __shared__ int s_seq[FW];
    auto tiles_of = [&](int s) -> long long {
        int r0, n, len, tiles, groups;
        if (s >= a.b.n_seqs)
            return 0;
        kv8_seq(a.b, s, a.err, r0, n, len);
        return n ? seq_tiles<GV>(p, n, len, tiles, groups) : 0;
    };
    auto block_scan = [&](long long c, long long &all) { // exclusive sum over the threads, and the sum
        long long x = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o)
                x += y;
        }
        __syncthreads();
        if (lane == 31)
            s_sum[warp] = x;
        __syncthreads();
        all = 0;
        long long before = 0;
#pragma unroll
        for (int w = 0; w < FW; w++) {
            before += w < warp ? s_sum[w] : 0;
            all += s_sum[w];
        }
        return before + x - c;
    };
    long long total = 0, all;
    const long long c0 = tiles_of(threadIdx.x), e0 = block_scan(c0, all);
    total = all;
    for (int s0 = FW * 32; s0 < a.b.n_seqs; s0 += FW * 32) {
        block_scan(tiles_of(s0 + threadIdx.x), all);
        total += all;
    }
    const int slots = gridDim.x * FW;
    const int active = (int)min((long long)slots, total);
    if (threadIdx.x < FW)
        s_seq[threadIdx.x] = 0;
    __syncthreads();
    long long base = 0;
    for (int s0 = 0; s0 < a.b.n_seqs; s0 += FW * 32) { // the sequence that holds each warp's first tile
        const int s = s0 + threadIdx.x;
        const long long c = s0 ? tiles_of(s) : c0;
        const long long e = base + (s0 ? block_scan(c, all) : e0);
        if (s0 == 0 && a.b.n_seqs > FW * 32)
            block_scan(c0, all);
        for (int w = 0; w < FW; w++) {
            const long long to = w * (long long)gridDim.x + blockIdx.x, u = to < active ? total * to / active : -1;
            if (u >= e && u < e + c) {
                s_seq[w] = s;
                s_at[w] = e;
            }
        }
        base += all;
    }
    __syncthreads();
    griddep_wait(); // the kernels for many rows are done with the workspace
    const int slot = warp * gridDim.x + blockIdx.x;
    const long long lo = slot < active ? total * slot / active : 0;
    const long long hi = slot < active ? total * (slot + 1) / active : 0;
    if (lane == 0)
        p.head[slot].pieces = 0;
    if (lo == hi)
        return;
    int win_s = s_seq[warp];
    long long win_base = s_at[warp]; // first tile of sequence win_s

    // ---- tile records, 32 at a time: lane i describes tile `from + i`
    int made = 0; // records made so far
    auto describe = [&]() {
        const long long from = lo + made;
        int r0 = 0, n = 0, len = 0, tiles = 0, groups = 0;
        long long c = 0, incl = 0;
        for (;;) { // the window of 32 sequences that holds `from`
            const int s = win_s + lane;
            n = 0;
            c = 0;
            if (s < a.b.n_seqs) {
                kv8_seq(a.b, s, a.err, r0, n, len);
                c = n ? seq_tiles<GV>(p, n, len, tiles, groups) : 0;
            }
            incl = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o)
                    incl += y;
            }
            const long long all = __shfl_sync(0xffffffffu, incl, 31);
            if (from < win_base + all || win_s + 32 >= a.b.n_seqs)
                break;
            win_base += all;
            win_s += 32;
        }
        const long long u = from + lane - win_base;
        int j = 0; // sequences of the window that end at or before u
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const long long e = __shfl_sync(0xffffffffu, incl, j + o - 1);
            if (e <= u)
                j += o;
        }
        const long long window = __shfl_sync(0xffffffffu, incl, 31);
        const bool here = from + lane < hi && u < window;
        const int jj = j & 31;
        const long long first = __shfl_sync(0xffffffffu, incl - c, jj);
        Tile x;
        x.s = win_s + jj;
        const int n_tiles = __shfl_sync(0xffffffffu, tiles, jj);
        x.len = __shfl_sync(0xffffffffu, len, jj);
        x.r0 = __shfl_sync(0xffffffffu, r0, jj);
        x.n = __shfl_sync(0xffffffffu, n, jj);
        const int ng = __shfl_sync(0xffffffffu, groups, jj);
        if (here) {
            const long long r = u - first;
            x.pair = (int)(r / n_tiles); // the groups of a KV head follow one another and share its codes in the L2
            x.tile = (int)(r - (long long)x.pair * n_tiles);
            const int g = x.pair / ng;
            const int t0 = x.tile * FT;
            auto piece = [&](int pos, int &row, float &ks, float &vs) {
                row = -1;
                ks = vs = 0.0f;
                if (pos >= x.len + x.n)
                    return;
                const int id = kv8_page(a.b, a.c, x.s, pos / page, a.err);
                if (id < 0)
                    return;
                const size_t at = (size_t)id * a.c.n_kv + g;
                row = (int)(at * page) + pos % page;
                ks = a.c.ks[at];
                vs = a.c.vs[at];
            };
            piece(t0, x.row0, x.ks0, x.vs0);
            if (page == 16) {
                piece(t0 + 16, x.row1, x.ks1, x.vs1);
            } else {
                x.row1 = x.row0;
                x.ks1 = x.ks0;
                x.vs1 = x.vs0;
            }
            const int4 *src = reinterpret_cast<const int4 *>(&x);
            int4 *dst = reinterpret_cast<int4 *>(&rec[(made + lane) % Lay::TILES]);
#pragma unroll
            for (int i = 0; i < 3; i++)
                dst[i] = src[i];
        }
        made += __popc(__ballot_sync(0xffffffffu, here));
        __syncwarp();
    };

    int mine = (int)(hi - lo);
    const uint64_t policy = policy_evict_first();
    auto issue = [&](int i, int v) { // lane 0: the K (v = 0) or V codes of tile i into stage i % ST
        const Tile &x = rec[i % Lay::TILES];
        uint8_t *dst = ring + ((i % ST) * 2 + v) * Lay::BOX;
        uint64_t *b = &bar[(i % ST) * 2 + v];
        const CUtensorMap *map = v ? &p.tv : &p.tk;
        const int row0 = x.row0, row1 = x.row1;
        if (page == 16) {
            mbar_arrive_expect_tx(b, ((row0 >= 0) + (row1 >= 0)) * (Lay::BOX / 2));
            if (row0 >= 0)
                tma_box(dst, map, row0, b, policy);
            if (row1 >= 0)
                tma_box(dst + Lay::BOX / 2, map, row1, b, policy);
        } else {
            mbar_arrive_expect_tx(b, row0 >= 0 ? Lay::BOX : 0);
            if (row0 >= 0)
                tma_box(dst, map, row0, b, policy);
        }
    };

    // ---- the pair in progress
    uint32_t qf[NT][KS][2];     // q as B fragments
    uint2 ql[NT][SPLIT || Lay::QLS ? 1 : KS]; // its small pieces, here or
    uint2 *qls = reinterpret_cast<uint2 *>(smem + Lay::ql_off) + warp * NT * KS * 32 + lane; // [column tile][k step][lane]
    float acc[MT][NT][4];       // O^T: (dim row gl / gl+8, column 2t4 / 2t4+1)
    float m[NT][2], l[NT][2], fac[NT][2];
    int lim[NT][2];             // last position the column's row attends to
    int pair_g = 0, pair_group = 0; // its KV head and group
    auto begin = [&](const Tile &x) {
        const int groups = (x.n * rep + GV - 1) / GV;
        pair_g = x.pair / groups;
        pair_group = x.pair - pair_g * groups;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const int v = pair_group * GV + (SPLIT ? 4 * j + (gl & 3) : 8 * j + gl);
            const int row = v / rep, head = pair_g * rep + v % rep;
            const bool live = row < x.n;
            float q[LD];
            float big = 0.0f;
            if (live) {
                const T *src = reinterpret_cast<const T *>(a.q) + (size_t)(x.r0 + row) * a.ld_q + (size_t)head * D;
                constexpr int H = D / 2;
                const int d0 = LD * t4, other = d0 ^ H;
                const float sign = d0 < H ? -1.0f : 1.0f;
                const size_t at = (size_t)(x.len + row) * H + (d0 & (H - 1));
#pragma unroll
                for (int i = 0; i < LD; i += 4) {
                    const float4 w = kv8_load4(src + d0 + i);
                    q[i] = w.x, q[i + 1] = w.y, q[i + 2] = w.z, q[i + 3] = w.w;
                    if (a.r.cos) {
                        const float4 o = kv8_load4(src + other + i), c = kv8_load4(a.r.cos + at + i),
                                     s = kv8_load4(a.r.sin + at + i);
                        // lower half: x c - y s; upper half: y s + x c
                        q[i] = __fadd_rn(__fmul_rn(w.x, c.x), sign * __fmul_rn(o.x, s.x));
                        q[i + 1] = __fadd_rn(__fmul_rn(w.y, c.y), sign * __fmul_rn(o.y, s.y));
                        q[i + 2] = __fadd_rn(__fmul_rn(w.z, c.z), sign * __fmul_rn(o.z, s.z));
                        q[i + 3] = __fadd_rn(__fmul_rn(w.w, c.w), sign * __fmul_rn(o.w, s.w));
                    }
                }
#pragma unroll
                for (int i = 0; i < LD; i++)
                    big = fmaxf(big, fabsf(q[i]));
            } else {
#pragma unroll
                for (int i = 0; i < LD; i++)
                    q[i] = 0.0f;
            }
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
            // a power of two brings the vector's largest value into [1, 2): f16 holds it with
            // its eleven bits whatever q's magnitude
            int e = (int)((__float_as_uint(big) >> 23) & 255u) - 127;
            e = max(-126, min(126, e));
            const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                uint32_t low[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float x0 = q[4 * k + 2 * h] * down, x1 = q[4 * k + 2 * h + 1] * down;
                    const uint32_t w = pack16(x0, x1);
                    const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&w));
                    low[h] = pack16(x0 - r.x, x1 - r.y);
                    qf[j][k][h] = SPLIT && gl >= 4 ? low[h] : w;
                }
                if constexpr (Lay::QLS) // read back by this lane alone
                    qls[(j * KS + k) * 32] = make_uint2(low[0], low[1]);
                else if constexpr (!SPLIT)
                    ql[j][k] = make_uint2(low[0], low[1]);
            }
            const float f = up * a.scale * 1.4426950408889634f; // scores in powers of two
            const int pos = live ? x.len + row : -1;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int from = (SPLIT ? (2 * t4 + c) & 3 : 2 * t4 + c) * 4;
                fac[j][c] = __shfl_sync(0xffffffffu, f, from);
                lim[j][c] = __shfl_sync(0xffffffffu, pos, from);
                m[j][c] = -INFINITY;
                l[j][c] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    acc[i][j][c] = 0.0f;
        }
    };

    int k_issued = 0, v_issued = 0; // tiles
    bool ok = true;
    auto arrived = [&](int i, int v) {
        if (ok)
            ok = kv8_wait(&bar[(i % ST) * 2 + v], (uint32_t)((i / ST) & 1), a.err);
        ok = __all_sync(0xffffffffu, ok);
        return ok;
    };
    auto refill = [&](int v, int &issued) { // the warp has read a stage
        __syncwarp();
        if (issued < mine) {
            if (lane == 0) {
                fence_proxy_async_smem(); // reads before the refill
                issue(issued, v);
            }
            issued++;
        }
    };
    auto consume = [&](const Tile &x, int at) {
        const uint8_t *kb = ring + (at % ST) * 2 * Lay::BOX, *vb = kb + Lay::BOX;
        if (!arrived(at, 0))
            return;
        float s[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; mt++) {
            // the lane's LD codes of tokens gl and gl + 8, in 16-byte units
#pragma unroll
            for (int u = 0; u < LD / 16; u++) {
                uint4 w[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int r = mt * 16 + h * 8 + gl;
                    const int unit = (LD / 16) * t4 + u;
                    const int sw = D == 128 ? unit ^ (r & 7) : unit ^ ((r >> 1) & 3);
                    w[h] = *reinterpret_cast<const uint4 *>(kb + r * D + sw * 16);
                }
                const uint32_t w0[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, w1[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t x0 = w0[k] ^ 0x80808080u, x1 = w1[k] ^ 0x80808080u;
                    const uint32_t a0 = codes_f16(x0, 0x4140), a2 = codes_f16(x0, 0x4342);
                    const uint32_t a1 = codes_f16(x1, 0x4140), a3 = codes_f16(x1, 0x4342);
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        const bool first = u == 0 && k == 0;
                        if constexpr (!SPLIT) {
                            const uint2 b = Lay::QLS ? qls[(j * KS + 4 * u + k) * 32] : ql[j][Lay::QLS ? 0 : 4 * u + k];
                            if (first)
                                mma16816_first(s[mt][j], a0, a1, a2, a3, b.x, b.y);
                            else
                                mma16816(s[mt][j], a0, a1, a2, a3, b.x, b.y);
                        }
                        if (SPLIT && first)
                            mma16816_first(s[mt][j], a0, a1, a2, a3, qf[j][0][0], qf[j][0][1]);
                        else
                            mma16816(s[mt][j], a0, a1, a2, a3, qf[j][4 * u + k][0], qf[j][4 * u + k][1]);
                    }
                }
            }
        }
        refill(0, k_issued);
        const float vs0 = x.vs0 * (1.0f / P_SCALE), vs1 = x.vs1 * (1.0f / P_SCALE);
        const bool half = page == 16;
        const int t0 = x.tile * FT;
        const bool whole = t0 + FT <= x.len + 1 && x.row0 >= 0 && x.row1 >= 0;
        uint32_t pf[2][NT][2]; // P as B fragments
        float corr[NT][2];
#pragma unroll
        for (int j = 0; j < NT; j++) {
            float tm[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                const float ks = mt ? x.ks1 : x.ks0;
                const bool there = (mt ? x.row1 : x.row0) >= 0;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    float y = s[mt][j][c];
                    if constexpr (SPLIT)
                        y += __shfl_xor_sync(0xffffffffu, y, 2);
                    y *= ks * fac[j][c & 1];
                    if (!whole && !(there && t0 + mt * 16 + (c >> 1) * 8 + gl <= lim[j][c & 1]))
                        y = -INFINITY;
                    s[mt][j][c] = y;
                    tm[c & 1] = fmaxf(tm[c & 1], y);
                }
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1)
                    tm[c] = fmaxf(tm[c], __shfl_xor_sync(0xffffffffu, tm[c], o));
                const float mn = fmaxf(m[j][c], tm[c]);
                const float ref = mn == -INFINITY ? 0.0f : mn; // nothing seen yet: every p is exp2(-inf)
                corr[j][c] = ex2(m[j][c] - ref);
                m[j][c] = mn;
                tm[c] = ref;
            }
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                float e[4];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    e[c] = ex2(s[mt][j][c] - tm[c & 1]);
                    sum[c & 1] += e[c];
                    e[c] *= P_SCALE;
                }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t w = pack16(e[2 * h], e[2 * h + 1]);
                    if constexpr (SPLIT) {
                        const float2 r = __half22float2(*reinterpret_cast<const __half2 *>(&w));
                        const uint32_t rest = pack16(e[2 * h] - r.x, e[2 * h + 1] - r.y);
                        w = t4 < 2 ? w : rest;
                    }
                    pf[mt][j][h] = transpose8x8(w);
                }
            }
#pragma unroll
            for (int c = 0; c < 2; c++)
                l[j][c] = l[j][c] * corr[j][c] + sum[c];
        }
        if (!arrived(at, 1))
            return;
        // O^T += V^T P: the tile's product in fresh accumulators, then one f32 step
        // a token's LV codes, tokens 2t4, 2t4+1, 2t4+8, 2t4+9 of each half
        constexpr int W = LV / 4; // 32-bit words
        uint32_t vw[2][4][W];
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = mt * 16 + 2 * t4 + (i & 1) + (i >> 1) * 8;
                if constexpr (D == 128) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(vb + r * D + ((gl ^ (r & 7)) << 4));
                    vw[mt][i][0] = w.x, vw[mt][i][1] = w.y, vw[mt][i][2] = w.z, vw[mt][i][3] = w.w;
                } else {
                    const uint2 w = *reinterpret_cast<const uint2 *>(
                        vb + r * D + (((gl >> 1) ^ ((r >> 1) & 3)) << 4) + (gl & 1) * 8);
                    vw[mt][i][0] = w.x, vw[mt][i][1] = w.y;
                }
            }
        refill(1, v_issued);
        // a new maximum scales what the sums hold (most tiles bring none to any column)
        bool moved = false;
#pragma unroll
        for (int j = 0; j < NT; j++)
            moved = moved || corr[j][0] != 1.0f || corr[j][1] != 1.0f;
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        acc[i][j][c] *= corr[j][c & 1];
        }
        auto add = [&](float (&o)[4], const float (&f)[4], float by) { // o += f * by
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                const float2 y = fma2(make_float2(f[c], f[c + 1]), make_float2(by, by), make_float2(o[c], o[c + 1]));
                o[c] = y.x;
                o[c + 1] = y.y;
            }
        };
#pragma unroll
        for (int k = 0; k < W; k++) {
            float f[2][NT][4];
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                // bytes (token, dim) -> per dim the token pairs (0, 1) and (2, 3)
                const uint32_t x01 = __byte_perm(vw[mt][0][k], vw[mt][1][k], 0x5140) ^ 0x80808080u;
                const uint32_t y01 = __byte_perm(vw[mt][0][k], vw[mt][1][k], 0x7362) ^ 0x80808080u;
                const uint32_t x23 = __byte_perm(vw[mt][2][k], vw[mt][3][k], 0x5140) ^ 0x80808080u;
                const uint32_t y23 = __byte_perm(vw[mt][2][k], vw[mt][3][k], 0x7362) ^ 0x80808080u;
                const uint32_t a0 = codes_f16(x01, 0x4140), a1 = codes_f16(x01, 0x4342);
                const uint32_t a2 = codes_f16(x23, 0x4140), a3 = codes_f16(x23, 0x4342);
                const uint32_t b0 = codes_f16(y01, 0x4140), b1 = codes_f16(y01, 0x4342);
                const uint32_t b2 = codes_f16(y23, 0x4140), b3 = codes_f16(y23, 0x4342);
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    if (mt == 0) {
                        mma16816_first(f[0][j], a0, a1, a2, a3, pf[0][j][0], pf[0][j][1]);
                        mma16816_first(f[1][j], b0, b1, b2, b3, pf[0][j][0], pf[0][j][1]);
                    } else {
                        mma16816(f[0][j], a0, a1, a2, a3, pf[1][j][0], pf[1][j][1]);
                        mma16816(f[1][j], b0, b1, b2, b3, pf[1][j][0], pf[1][j][1]);
                    }
                }
                if (half && mt == 0) { // pages of 16: the two halves have scales of their own
#pragma unroll
                    for (int i = 0; i < 2; i++)
#pragma unroll
                        for (int j = 0; j < NT; j++) {
                            add(acc[2 * k + i][j], f[i][j], vs0);
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                f[i][j][c] = 0.0f;
                        }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < NT; j++)
                    add(acc[2 * k + i][j], f[i][j], vs1);
        }
    };

    // the pair's segment is over: write it out, or keep it as a piece
    auto finish = [&](const Tile &x, bool from_start, bool to_end) {
        const bool done = from_start && to_end;
        const int which = from_start ? 1 : 0;
        float *part = p.part + ((size_t)slot * 2 + which) * GV * (D + 2);
        if (from_start && !to_end && lane == 0) { // hi - 1 is tile x.tile; the range that holds the pair's last one
            const long long end = hi - 1 + (x.n_tiles() - 1 - x.tile);
            JoinHead h{};
            h.pieces = (int)(((end + 1) * active - 1) / total) - slot + 1;
            h.first = pair_group * GV;
            h.vectors = min(GV, x.n * rep - h.first);
            h.g = pair_g;
            h.r0 = x.r0;
            p.head[slot] = h;
        }
#pragma unroll
        for (int j = 0; j < NT; j++) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float sum = l[j][c];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1)
                    sum += __shfl_xor_sync(0xffffffffu, sum, o);
                float o[LV]; // dims LV*gl ..
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float y = acc[i][j][2 * h + c];
                        if constexpr (SPLIT)
                            y += __shfl_xor_sync(0xffffffffu, y, 2);
                        o[2 * i + h] = y;
                    }
                const int vi = SPLIT ? 4 * j + 2 * t4 + c : 8 * j + 2 * t4 + c; // vector within the group
                const int v = pair_group * GV + vi;
                if ((SPLIT && t4 >= 2) || v >= x.n * rep)
                    continue;
                if (done) {
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                    for (int i = 0; i < LV; i++)
                        o[i] *= inv;
                    T *out = reinterpret_cast<T *>(a.out) + (size_t)(x.r0 + v / rep) * a.ld_out +
                             (size_t)(pair_g * rep + v % rep) * D + LV * gl;
                    store_row<LV>(out, o);
                } else {
                    float *dst = part + (size_t)vi * D + LV * gl;
                    store_row<LV>(dst, o);
                    if (gl == 0) {
                        part[(size_t)GV * D + vi] = m[j][c];
                        part[(size_t)GV * (D + 1) + vi] = sum;
                    }
                }
            }
        }
    };

    auto describe_to = [&](int least) { // records of the range's first `least` tiles, at the least
        while (made < min(mine, least)) {
            const int before = made;
            describe();
            if (made == before) // only if the batch's numbers changed under way
                mine = made;
        }
    };
    describe_to(ST);
    k_issued = v_issued = min(mine, ST);
    if (lane == 0)
        for (int i = 0; i < k_issued; i++) {
            issue(i, 0);
            issue(i, 1);
        }
    bool from_start = false;
    int done = 0; // tiles consumed
    for (; done < mine; done++) {
        // records ahead of the loads
        describe_to(done + Lay::TILES - Lay::BATCH + 1);
        const Tile x = rec[done % Lay::TILES];
        if (done == 0 || x.tile == 0) {
            from_start = x.tile == 0;
            begin(x);
        }
        consume(x, done);
        if (!ok)
            break;
        const bool to_end = x.tile == x.n_tiles() - 1;
        if (to_end || done == mine - 1)
            finish(x, from_start, to_end);
    }
    if (!ok && lane == 0) // copies in flight land before the shared memory goes
        for (int i = done; i < k_issued; i++)
            for (int v = 0; v < 2 && (v == 0 || i < v_issued); v++)
                for (int it = 0; it < 100000 && !mbar_try_wait(&bar[(i % ST) * 2 + v], (uint32_t)((i / ST) & 1)); it++)
                    ;
}

// a code pool as rows of D bytes in swizzled boxes of `rows` rows
int encode_codes(CUtensorMap *map, const int8_t *codes, const Kv8 &c, int rows)
{
    auto fn = tensor_map_encoder();
    if (!fn)
        return fail(LLMRS_ECUDA, "cuTensorMapEncodeTiled unavailable");
    cuuint64_t dims[2] = {(cuuint64_t)c.D, (cuuint64_t)c.n_pages * c.n_kv * c.page};
    cuuint64_t strides[1] = {(cuuint64_t)c.D};
    cuuint32_t box[2] = {(cuuint32_t)c.D, (cuuint32_t)rows};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(codes), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE,
                          c.D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(LLMRS_ECUDA, "cuTensorMapEncodeTiled (code pool) failed (%d)", (int)r);
    return LLMRS_OK;
}

template <class T, int D, bool SPLIT, int NT>
int run_few(const FewParams &p, int ctas, cudaStream_t stream)
{
    constexpr int GV = group_vectors<SPLIT, NT>();
    constexpr int FW = few_warps(NT);
    LLMRS_CUDA_TRY(launch(kv8_few_kernel<T, D, SPLIT, NT>, dim3(ctas), dim3(FW * 32), FewLay<D, SPLIT, NT>::bytes, stream,
                          p.many != INT32_MAX, p));
    LLMRS_CUDA_TRY(launch(kv8_join_kernel<T, D, GV>, dim3(4 * ctas), dim3(JT), 0, stream, true, p.a,
                          (const float *)p.part, (const JoinHead *)p.head, ctas * FW));
    return LLMRS_OK;
}

template <class T, int D, bool SPLIT>
int run_nt(const FewParams &p, int nt, int ctas, cudaStream_t stream)
{
    if (nt == 1)
        return run_few<T, D, SPLIT, 1>(p, ctas, stream);
    return run_few<T, D, SPLIT, 2>(p, ctas, stream);
}

template <class T, bool SPLIT>
int run_d(const FewParams &p, int nt, int ctas, cudaStream_t stream)
{
    return p.a.c.D == 128 ? run_nt<T, 128, SPLIT>(p, nt, ctas, stream) : run_nt<T, 64, SPLIT>(p, nt, ctas, stream);
}

template <class T, bool SPLIT, int D, int NT>
cudaError_t prepare_few()
{
    return cudaFuncSetAttribute(kv8_few_kernel<T, D, SPLIT, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                FewLay<D, SPLIT, NT>::bytes);
}

template <class T, bool SPLIT>
cudaError_t prepare_all()
{
    cudaError_t e = prepare_few<T, SPLIT, 128, 1>();
    if (e == cudaSuccess)
        e = prepare_few<T, SPLIT, 128, 2>();
    if (e == cudaSuccess)
        e = prepare_few<T, SPLIT, 64, 1>();
    if (e == cudaSuccess)
        e = prepare_few<T, SPLIT, 64, 2>();
    return e;
}

// columns / 8 for the average sequence's vectors per KV head: a longer sequence
// takes several groups, and each reads the codes again (from the L2, mostly).
// 32 columns at a head of 128 do not fit the registers (f32 rows, 16 sequences
// of 300 to 4000 tokens, 16 vectors each: 96 us against 68 for two groups).
int few_nt(long long vectors, int per)
{
    return vectors <= per ? 1 : 2;
}

long long mean_vectors(int rep, int n_rows, int n_seqs)
{
    return n_seqs > 0 ? ((long long)n_rows + n_seqs - 1) / n_seqs * rep : 0;
}

// A sequence with more vectors per KV head than this goes to the kernel for many
// rows: three groups here cost what its tile of 128 rows costs whatever it holds.
// 16 sequences of 300 to 4000 tokens, heads of 128, f32 rows: 16 vectors 68 us
// here, 88 there, 32 vectors 109 and 90; bf16 rows, both kernels launched: 16 vectors 57
// and 64, 32 vectors 75 and 66, 48 vectors 95 and 68, but sequences of 4 to 36 vectors
// side by side 68, and 78 with a border at 32; heads of 64 cross at the same places.
constexpr int many_from(int dtype) { return 3 * (dtype == LLMRS_BF16 ? 16 : 8); }

// whether a sequence may have that many: with no more rows than sequences (a
// decode step) every sequence is taken to have few, which is right for any
bool some_many(int rep, int n_rows, int n_seqs, int from)
{
    return rep <= MANY_MAX_REP && n_rows > n_seqs && (long long)n_rows * rep > from;
}

} // namespace

size_t kv8_attention_workspace(int n_heads, int n_kv, int head_dim, int n_rows, int n_seqs)
{
    const int rep = n_heads / n_kv;
    // two pieces a warp, of the vectors of a group (16-bit rows: eight to a column tile)
    size_t few = 0;
    for (int nt = 1; nt <= few_nt(mean_vectors(rep, n_rows, n_seqs), 4); nt++)
        few = std::max(few, JOIN_SLOTS * sizeof(JoinHead) + F_MAX_CTAS * 2 * (size_t)few_warps(nt) * 8 * nt *
                                                                (head_dim + 2) * sizeof(float));
    return some_many(rep, n_rows, n_seqs, many_from(LLMRS_F32)) ? std::max(few, kv8_many_workspace(head_dim, n_heads, n_rows)) : few;
}

int kv8_prepare(void)
{
    cudaError_t e = prepare_all<float, true>();
    if (e == cudaSuccess)
        e = prepare_all<__half, true>();
    if (e == cudaSuccess)
        e = prepare_all<__nv_bfloat16, false>();
    if (e != cudaSuccess)
        return fail(LLMRS_ECUDA, "kv8 kernel attributes: %s", cudaGetErrorString(e));
    return kv8_many_prepare();
}

int kv8_attention(const Kv8Attn &a, void *ws, int sms, cudaStream_t stream)
{
    const int rep = a.n_heads / a.c.n_kv;
    const int from = many_from(a.dtype);
    const bool both = some_many(rep, a.b.n_rows, a.b.n_seqs, from);
    if (both)
        LLMRS_TRY(kv8_many(a, from, ws, sms, stream));
    FewParams p{};
    p.a = a;
    LLMRS_TRY(encode_codes(&p.tk, a.c.kq, a.c, std::min(a.c.page, FT)));
    LLMRS_TRY(encode_codes(&p.tv, a.c.vq, a.c, std::min(a.c.page, FT)));
    p.head = reinterpret_cast<JoinHead *>(ws);
    p.part = reinterpret_cast<float *>(p.head + JOIN_SLOTS);
    p.many = both ? from : INT32_MAX;
    const int nt = few_nt(mean_vectors(rep, a.b.n_rows, a.b.n_seqs), a.dtype == LLMRS_BF16 ? 8 : 4);
    const int ctas = std::min(sms, F_MAX_CTAS);
    if (a.dtype == LLMRS_F32)
        return run_d<float, true>(p, nt, ctas, stream);
    if (a.dtype == LLMRS_BF16)
        return run_d<__nv_bfloat16, false>(p, nt, ctas, stream);
    return run_d<__half, true>(p, nt, ctas, stream);
}

} // namespace llmrs
