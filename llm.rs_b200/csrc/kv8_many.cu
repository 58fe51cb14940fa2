// kv8_many.cu - causal attention over the paged 8-bit KV cache for many rows
// per sequence (prompts, chunks of them): tcgen05 tensor cores (sm_100a).
//
// A CTA's tile is 128 vectors (row, query head) of one KV head by 128 tokens:
//   S = Q K^T (128 x 128, K = D), P = exp2(S * ks - max) * vs, O = P V,
// f16 operands, f32 accumulators in TMEM.  The codes are exact in f16.  f32
// rows: Q and P are two f16 pieces each (22 bits and more), so the products
// run twice; f16 rows too (with P in one piece they are 1.4 times as far off as
// the rounding of the result); bf16 rows: two of Q, whose errors a sharp head's
// softmax multiplies, and one of P, 11 bits to the result's 8.  The two prompts below,
// 2-norm error and time: 1.66e-3, the rounding of the result alone, and 530 us; with
// value scales' mantissas in P 1.67e-3 and 523 us, with one piece of Q too 1.72e-3 (and
// several times the rounding where scores reach some tens) and 475; with two of P 1.66e-3
// and 615.  Every tile's O is a fresh product that registers add up in f32, with the
// change of the maximum applied there: long sums do not pass through the tensor core's
// accumulator.
//
// Warpgroups: 0 and 4 softmax of every other tile (thread = row), 1 output
// (thread = row, D accumulators), 2 and 5 key and value codes to f16 in shared
// memory (keys K-major, values MN-major, both 128-byte swizzled: the same image),
// 3: one warp issues the products, one looks up pages and scales ahead, one
// fetches Q, which a kernel of its own has rotated, scaled and split.
// The softmax keeps no state: it hands over a tile's maximum, sum and scale, and
// the output warps, which go through the tiles in order, know the running ones.
// TMEM: three S, P over the S it came from, and O in the rest (once for heads of
// 128, twice for 64): tiles i and i + 1 are in the softmax while the product of
// tile i - 1 runs and the scores of tile i + 2 are made.  K and V are double
// buffered, Q too but for two pieces of 128 dims.
//
// What a tile costs is not its products' 1000 to 2000 cycles but the roles' chains, whose
// instructions take 4 to 5 cycles each: so each role that was the longest got a
// second warpgroup or a kernel of its own, and each keeps its next loads (TMEM
// columns, codes) in flight while it works.  Two prompts of 3500 to 4096 rows,
// bf16, 32 heads of 128 over 8: 530 us (462 TFLOP/s; with one piece of Q 475, and
// 740 with one softmax, one widening and one Q warpgroup), chunks of 3 prompts of
// 1000 rows behind 0 to 3000 tokens, f32: 267 us.  Left: 3400 to 3900 cycles a tile,
// spread over all roles: of 493 us (an earlier build, one piece of Q) 394 stayed
// without any softmax, 454 without widening, 471 without the output's sums.
//
// Work: the tiles of all (sequence, KV head, tile of rows) in one row, cut into
// equal consecutive ranges, one per CTA; pieces of a softmax that a range cuts
// are joined by a second kernel (kv8_core.cuh).
#include <limits.h>

#include "gemv.cuh"
#include "kv8_core.cuh"
#include "kv8_many.cuh"

namespace llmrs {

namespace {

constexpr int MB = 128;          // vectors, and tokens, of a tile
constexpr int MANY_THREADS = 768;
constexpr int INFO = 8;          // tile descriptions in flight
// softmax -> output hand-overs in flight: the scores of tile i wait for the product of
// tile i - NS, and that for the output to have taken one or two tiles before it
constexpr int RING = 6;
constexpr int NS = 3;            // buffers of S
constexpr int QT = 256;          // threads of the kernel that prepares Q

struct ManyTile {
    int row[8];                  // pool rows of the tile's 16-token groups; -1: not there
    float ks[8];                 // key scales
    float vs[8];                 // value scales
    float lvs[8];                // log2 of them, rounded up (-inf: zero)
    int first, last, masked;     // of the pair within this range; some row does not see all tokens
    int tile;                    // of tokens
    int pad0;                    // g at 8 of 16 bytes: at 4 the kernel spills 76 bytes, not 16 (7 %)
    int g, mt;                   // KV head, tile of rows
    int r0, n, len;              // of the sequence
    int from_start, to_end, pieces;
    int item;                    // number of the pair within this range
    int pad1[2];
};
static_assert(sizeof(ManyTile) == 192, "16-byte words");

struct ManyParams {
    CUtensorMap tq;   // prepared Q: [piece][row][head][D] f16, boxes of 64 dims of a tile's vectors
    Kv8Attn a;
    __half *q16;      // the same memory
    float *facs;      // [row][head] what the scores are multiplied by
    float *part;
    JoinHead *head;
    int many; // sequences with at most this many vectors per KV head are another kernel's
};

template <int D, int QP>
struct ManyLay {
    static constexpr int KVS = 2;                   // buffers of K and of V
    static constexpr int QS = QP * D > 128 ? 1 : 2; // of Q
    static constexpr int OS = (512 - NS * MB) / D;  // of O
    static constexpr int T = MB * D * 2;        // bytes of one piece of Q, of an f16 K or V tile
    static constexpr int k_off = QS * QP * T;   // Q: [buffers][QP pieces]
    static constexpr int v_off = k_off + KVS * T;
    static constexpr int info_off = v_off + KVS * T;
    static constexpr int ring_off = info_off + INFO * (int)sizeof(ManyTile);
    static constexpr int bar_off = ring_off + RING * 3 * MB * 4;
    static constexpr int bytes = bar_off + 512 + 1024; // + alignment slack
    static_assert(bytes <= 232448 - 256, "shared memory of one CTA");
};

enum : int { // barriers
    B_INFO_FULL = 0,
    B_INFO_EMPTY = B_INFO_FULL + INFO,
    B_K_FULL = B_INFO_EMPTY + INFO,
    B_K_EMPTY = B_K_FULL + 2,
    B_V_FULL = B_K_EMPTY + 2,
    B_V_EMPTY = B_V_FULL + 2,
    B_S_FULL = B_V_EMPTY + 2,
    B_P_FULL = B_S_FULL + NS,
    B_P_EMPTY = B_P_FULL + NS,
    B_O_FULL = B_P_EMPTY + NS,
    B_O_EMPTY = B_O_FULL + 2,
    B_Q_FULL = B_O_EMPTY + 2,
    B_Q_EMPTY = B_Q_FULL + 2,
    B_COUNT = B_Q_EMPTY + 2,
};
static_assert(B_COUNT * 8 <= 512, "barrier space");

// ------------------------------------------------------------ tcgen05
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tc_commit(uint64_t *bar)
{
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar))
                 : "memory");
}

// Operand tile in 128-byte-swizzled atoms of 8 rows x 128 bytes, 1024 bytes
// apart.  K-major: rows are M or N, 64 K values each (lead unused).  MN-major:
// rows are K, 64 M or N values each, `lead` bytes to the next 64.  The low word
// of its descriptor, whose unit is 16 bytes; the high word is always the same.
__device__ __forceinline__ uint32_t sw128(uint32_t saddr, uint32_t lead) { return (saddr >> 4) | (lead >> 4) << 16; }
constexpr uint32_t SW128_HI = (1024u >> 4) | 1u << (46 - 32) | 2u << (61 - 32);

// kind::f16: f16 x f16 -> f32, M = 128; B K-major or MN-major
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_mn)
{
    return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(MB >> 4) << 24);
}

// Four steps of 16 along K, 32 bytes apart in both operands.  Whole warp, one
// elected lane issues, and the descriptors are sums of low words in one block:
// in a divergent branch, or with a descriptor built per step, a step took 140
// to 200 cycles to issue, and 64 to run.
__device__ __forceinline__ void mma_ss4(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool acc)
{
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b32 x, y;\n\t.reg .b64 da, db;\n\t"
                 "elect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t"
                 "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 da, {x, %3};\n\tmov.b64 db, {y, %3};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, 1;\n\t"
                 "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 da, {x, %3};\n\tmov.b64 db, {y, %3};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, 1;\n\t"
                 "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 da, {x, %3};\n\tmov.b64 db, {y, %3};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, 1;\n\t}" ::"r"(d),
                 "r"(a_lo), "r"(b_lo), "n"(SW128_HI), "r"(idesc), "r"((int)acc)
                 : "memory");
}

// the same with A in TMEM, 16 columns a step, and B MN-major, 16 rows of 128 bytes a step
__device__ __forceinline__ void mma_ts4(uint32_t d, uint32_t at, uint32_t b_lo, uint32_t idesc, bool acc)
{
    asm volatile("{\n\t.reg .pred p, q;\n\t.reg .b32 x, y;\n\t.reg .b64 db;\n\t"
                 "elect.sync _|q, 0xffffffff;\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "mov.b64 db, {%2, %3};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t"
                 "add.u32 x, %1, 16;\n\tadd.u32 y, %2, 128;\n\tmov.b64 db, {y, %3};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %4, 1;\n\t"
                 "add.u32 x, %1, 32;\n\tadd.u32 y, %2, 256;\n\tmov.b64 db, {y, %3};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %4, 1;\n\t"
                 "add.u32 x, %1, 48;\n\tadd.u32 y, %2, 384;\n\tmov.b64 db, {y, %3};\n\t"
                 "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %4, 1;\n\t}" ::"r"(d),
                 "r"(at), "r"(b_lo), "n"(SW128_HI), "r"(idesc), "r"((int)acc)
                 : "memory");
}

#define R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), \
                 "=r"(r[o + 6]), "=r"(r[o + 7])
#define T8(r, o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), \
                 "+r"(r[o + 6]), "+r"(r[o + 7])
#define I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), \
                 "r"(r[o + 6]), "r"(r[o + 7])

// 32 consecutive columns of this thread's TMEM lane; tm_wait makes them usable
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24)
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tm_wait(uint32_t (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : T8(r, 0), T8(r, 8), T8(r, 16), T8(r, 24) : : "memory");
}
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t (&r)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::I8(r, 0),
                 I8(r, 8), I8(r, 16), I8(r, 24), "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15}, [%16];"
                 : R8(r, 0), R8(r, 8)
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void tm_wait(uint32_t (&r)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : T8(r, 0), T8(r, 8) : : "memory");
}
__device__ __forceinline__ void tm_st8(uint32_t addr, const uint32_t (&r)[8])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::I8(r, 0), "r"(addr)
                 : "memory");
}
#undef R8
#undef T8
#undef I8

// 2^n, -126 <= n <= 126
__device__ __forceinline__ float exp2i(int n) { return __int_as_float((n + 127) << 23); }

// whether a barrier's phase is over, without waiting
__device__ __forceinline__ bool mbar_test(uint64_t *bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(smem_addr(bar)), "r"(parity)
                 : "memory");
    return ok != 0;
}

template <int N>
__device__ __forceinline__ void regs_up()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// ------------------------------------------------------------ the tiles of a sequence
// Tile of rows mt holds rows [mt*R, (mt+1)*R), whole rows of rep vectors each;
// vector r of it is row mt*R + r / rep, head r % rep.  It needs the tokens up
// to its last row's position.
__device__ __forceinline__ int row_tiles(int n, int R) { return (n + R - 1) / R; }
__device__ __forceinline__ int token_tiles(int len, int n, int R, int mt) { return (len + min(n, (mt + 1) * R) - 1) / MB + 1; }

__device__ __forceinline__ long long head_tiles(int len, int n, int R)
{
    long long t = 0;
    for (int mt = 0, m = row_tiles(n, R); mt < m; mt++)
        t += token_tiles(len, n, R, mt);
    return t;
}

// The (sequence, KV head, tile of rows) pairs in their order
struct Walk {
    int s, r0, n, len, g, mt, nt; // nt: tiles of tokens
    __device__ __forceinline__ int start(const ManyParams &p, int s_, long long off, int R) // returns the tile at `off`
    {
        s = s_;
        kv8_seq(p.a.b, s, p.a.err, r0, n, len);
        const long long ht = head_tiles(len, n, R);
        g = (int)(off / ht);
        off -= g * ht;
        for (mt = 0; off >= (nt = token_tiles(len, n, R, mt)); mt++)
            off -= nt;
        return (int)off;
    }
    __device__ __forceinline__ void next(const ManyParams &p, int rep, int R)
    {
        if (++mt == row_tiles(n, R)) {
            mt = 0;
            if (++g == p.a.c.n_kv) {
                g = 0;
                do {
                    s++;
                    kv8_seq(p.a.b, s, p.a.err, r0, n, len);
                } while ((long long)n * rep <= p.many && s + 1 < p.a.b.n_seqs);
            }
        }
        nt = token_tiles(len, n, R, mt);
    }
};

// codes of 16 dims to f16, 32 bytes
__device__ __forceinline__ void widen(uint4 w, uint4 &lo, uint4 &hi)
{
    const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u, z = w.z ^ 0x80808080u, t = w.w ^ 0x80808080u;
    lo = make_uint4(codes_f16(x, 0x4140), codes_f16(x, 0x4342), codes_f16(y, 0x4140), codes_f16(y, 0x4342));
    hi = make_uint4(codes_f16(z, 0x4140), codes_f16(z, 0x4342), codes_f16(t, 0x4140), codes_f16(t, 0x4342));
}

// QP, PP: f16 pieces of Q and of P
template <class T, int D, int QP, int PP>
__global__ void __launch_bounds__(MANY_THREADS, 1) kv8_many_kernel(const __grid_constant__ ManyParams p)
{
    using Lay = ManyLay<D, QP>;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    ManyTile *info = reinterpret_cast<ManyTile *>(smem + Lay::info_off);
    float *ring = reinterpret_cast<float *>(smem + Lay::ring_off); // [RING][maximum | scale of O | sum][MB]
    uint64_t *bar = reinterpret_cast<uint64_t *>(smem + Lay::bar_off);
    __shared__ uint32_t s_tmem;
    __shared__ long long s_sum[MANY_THREADS / 32];
    __shared__ long long s_at;
    __shared__ int s_seq;
    const Kv8Attn &a = p.a;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, wg = warp >> 2;
    const int rep = a.n_heads / a.c.n_kv, R = MB / rep;
    griddep_launch_dependents();

    if (threadIdx.x == 0) {
        for (int i = 0; i < INFO; i++) {
            mbar_init(&bar[B_INFO_FULL + i], 1);
            mbar_init(&bar[B_INFO_EMPTY + i], 17); // 16 warps and the issuing thread
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar[B_K_FULL + i], 128);
            mbar_init(&bar[B_K_EMPTY + i], 1);
            mbar_init(&bar[B_V_FULL + i], 128);
            mbar_init(&bar[B_V_EMPTY + i], 1);
            mbar_init(&bar[B_O_FULL + i], 1);
            mbar_init(&bar[B_O_EMPTY + i], 128);
            mbar_init(&bar[B_Q_FULL + i], 1);
            mbar_init(&bar[B_Q_EMPTY + i], 1);
        }
        for (int i = 0; i < NS; i++) {
            mbar_init(&bar[B_S_FULL + i], 1);
            mbar_init(&bar[B_P_FULL + i], 128);
            mbar_init(&bar[B_P_EMPTY + i], 1);
        }
        fence_mbar_init();
        s_seq = 0;
    }

    // ---- this CTA's range of tiles
    auto tiles_of = [&](int s) -> long long {
        int r0, n, len;
        if (s >= a.b.n_seqs)
            return 0;
        kv8_seq(a.b, s, a.err, r0, n, len);
        return (long long)n * rep > p.many ? a.c.n_kv * head_tiles(len, n, R) : 0;
    };
    auto block_scan = [&](long long c, long long &all) {
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
        for (int w = 0; w < MANY_THREADS / 32; w++) {
            before += w < warp ? s_sum[w] : 0;
            all += s_sum[w];
        }
        return before + x - c;
    };
    long long total, all;
    const long long c0 = tiles_of(threadIdx.x), e0 = block_scan(c0, all), all0 = all;
    total = all;
    for (int s0 = MANY_THREADS; s0 < a.b.n_seqs; s0 += MANY_THREADS) {
        block_scan(tiles_of(s0 + threadIdx.x), all);
        total += all;
    }
    const int slot = blockIdx.x, active = (int)min((long long)gridDim.x, total);
    const long long lo = slot < active ? total * slot / active : 0;
    const long long hi = slot < active ? total * (slot + 1) / active : 0;
    if (threadIdx.x == 0)
        p.head[slot].pieces = 0;
    if (lo == hi)
        return;
    long long base = 0;
    for (int s0 = 0; s0 < a.b.n_seqs; s0 += MANY_THREADS) {
        const long long c = s0 ? tiles_of(s0 + threadIdx.x) : c0;
        const long long e = base + (s0 ? block_scan(c, all) : e0);
        if (lo >= e && lo < e + c) {
            s_seq = s0 + threadIdx.x;
            s_at = lo - e;
        }
        base += s0 ? all : all0;
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before();
    }
    __syncthreads();
    tc_after();
    const uint32_t tmem = s_tmem;
    const int mine = (int)(hi - lo);
    griddep_wait(); // Q is ready
    auto wait = [&](int b, int use) { // whole warp
        return __all_sync(0xffffffffu, kv8_wait(&bar[b], (uint32_t)(use & 1), a.err));
    };
    // Every role ends on its own, and no value in a register outlives one: behind the ends
    // roles with 48 and with 160 registers would meet.  After a wait that ran out, products in
    // flight end before their memory goes.
    auto leave = [&](bool ok) {
        for (int i = 0; i < 64 && !ok; i++)
            __nanosleep(1000);
        tc_before();
        asm volatile("bar.sync 1, %0;" ::"n"(MANY_THREADS) : "memory");
        tc_after();
    };

    if (wg == 0 || wg == 4) {
        bool ok = true;
        // ================================================= softmax of every other tile: thread = row
        static_assert(2 * 80 + 160 + 2 * 56 + 48 == 6 * 80, "the launch's registers, shared out");
        const int r = threadIdx.x & 127, odd = wg >> 2;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        float fac = 0.0f;
        int lim = -1, item = -1;
        bool busy = false; // some row of this warp is there
        for (int i = odd; i < mine && ok; i += 2) {
            const ManyTile &x = info[i % INFO];
            if (!(ok = wait(B_INFO_FULL + i % INFO, i / INFO) && wait(B_S_FULL + i % NS, i / NS)))
                break;
            tc_after();
            const uint32_t sp = lanes + (uint32_t)(i % NS) * MB;
            if (x.item != item) {
                item = x.item;
                const int row = x.mt * R + r / rep;
                const bool live = r < R * rep && row < x.n;
                lim = live ? x.len + row : -1;
                busy = __any_sync(0xffffffffu, live);
                fac = live ? p.facs[(size_t)(x.r0 + row) * a.n_heads + x.g * rep + r % rep] : 0.0f;
            }
            float top = -INFINITY, sum = 0.0f;
            int shift = 0; // P is p * vs * 2^shift / unit
            float unit = 1.0f;
            if (busy) {
                const bool masked = x.masked;
                if (masked) { // S becomes the scores themselves, the unseen ones at -inf
#pragma unroll 1
                    for (int k = 0; k < 4; k++) {
                        uint32_t s[32];
                        tm_ld32(sp + 32 * k, s);
                        tm_wait(s);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int last = x.row[2 * k + h] >= 0 ? lim - x.tile * MB - 32 * k - 16 * h : -1;
                            const float kf = fac * x.ks[2 * k + h];
#pragma unroll
                            for (int j = 0; j < 16; j++)
                                s[16 * h + j] =
                                    __float_as_uint(j <= last ? __uint_as_float(s[16 * h + j]) * kf : -INFINITY);
                        }
                        tm_st32(sp + 32 * k, s);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                const float f = masked ? 1.0f : fac;
                // the row's largest score, and a bound of the largest with its value scale
                float ref2 = -INFINITY;
                auto most = [&](int g, const uint32_t *s) { // 16 scores of group g
                    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        t0 = fmaxf(fmaxf(t0, __uint_as_float(s[j])), __uint_as_float(s[j + 1]));
                        t1 = fmaxf(fmaxf(t1, __uint_as_float(s[j + 2])), __uint_as_float(s[j + 3]));
                    }
                    t0 = fmaxf(t0, t1) * (masked ? 1.0f : f * x.ks[g]); // the factor is not negative
                    top = fmaxf(top, t0);
                    if constexpr (PP == 1)
                        unit = t0 + x.lvs[g] > ref2 ? x.vs[g] : unit;
                    ref2 = fmaxf(ref2, t0 + x.lvs[g]);
                };
                { // the next columns are on their way meanwhile
                    uint32_t s0[16], s1[16];
                    tm_ld16(sp, s0);
                    tm_wait(s0);
#pragma unroll 1
                    for (int g = 0; g < 8; g += 2) {
                        tm_ld16(sp + 16 * g + 16, s1);
                        most(g, s0);
                        tm_wait(s1);
                        tm_ld16(sp + min(16 * g + 32, 112), s0); // the last one is not used
                        most(g + 1, s1);
                        tm_wait(s0);
                    }
                }
                // P = p * vs, shifted so that the row's largest lies at 2^14: f16 keeps its bits
                // whatever the scales of pages that the row hardly sees.  p and vs are f32
                // factors, not one power of two, so P and the sum share p's rounding.
                const float ref = top == -INFINITY ? 0.0f : top;
                // P in one piece: the mantissa of the largest's scale goes back in with the output, so
                // that tokens of its pages have P = p * 2^n and a probability of one is exact
                float inv = 1.0f;
                if constexpr (PP == 1) {
                    unit = __uint_as_float((__float_as_uint(unit) & 0x7fffffu) | 0x3f800000u);
                    inv = __frcp_rn(unit);
                }
                if (ref2 > -INFINITY) // some seen page has a scale above 0
                    shift = (int)fminf(fmaxf(P_SCALE_LOG2 - ceilf(ref2 - ref), -126.0f), 126.0f);
                auto probabilities = [&](int g, const uint32_t *s) { // 16 of them, over the scores of group g
                    // where vs * 2^shift alone would overflow (its scores are far below the row's
                    // largest), 2^up goes to p
                    const float up = fmaxf(x.lvs[g] + (float)(shift - 60), 0.0f);
                    const float kf = masked ? 1.0f : f * x.ks[g], add = up - ref;
                    float by = x.vs[g] * exp2i(shift - (int)up);
                    if constexpr (PP == 1) { // by / unit, rounded once
                        const float q = by * inv;
                        by = fmaf(fmaf(-q, unit, by), inv, q);
                    }
                    float2 g01 = make_float2(0.0f, 0.0f);
                    uint32_t ph[8], pl[8];
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const float2 y = fma2(make_float2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])),
                                              make_float2(kf, kf), make_float2(add, add));
                        const float2 e = make_float2(ex2(y.x), ex2(y.y));
                        g01 = add2(g01, e);
                        const float2 o = mul2(e, make_float2(by, by));
                        const uint32_t w = pack16(o.x, o.y);
                        ph[j / 2] = w;
                        if constexpr (PP == 2) {
                            const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&w));
                            pl[j / 2] = pack16(o.x - h.x, o.y - h.y);
                        }
                    }
                    sum += up > 0.0f ? (g01.x + g01.y) * ex2(-up) : g01.x + g01.y;
                    tm_st8(sp + 16 * g, ph);
                    if constexpr (PP == 2)
                        tm_st8(sp + 16 * g + 8, pl);
                };
                {
                    uint32_t s0[16], s1[16];
                    tm_ld16(sp, s0);
                    tm_wait(s0);
#pragma unroll 1
                    for (int g = 0; g < 8; g += 2) {
                        tm_ld16(sp + 16 * g + 16, s1);
                        probabilities(g, s0);
                        tm_wait(s1);
                        tm_ld16(sp + min(16 * g + 32, 112), s0); // the last one is not used
                        probabilities(g + 1, s1);
                        tm_wait(s0);
                    }
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            }
            float *hand = ring + (i % RING) * 3 * MB;
            hand[r] = top;
            hand[MB + r] = exp2i(-shift) * unit;
            hand[2 * MB + r] = sum;
            tc_before();
            mbar_arrive(&bar[B_P_FULL + i % NS]);
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&bar[B_INFO_EMPTY + i % INFO]);
        }
        leave(ok);
    } else if (wg == 1) {
        // ================================================= output: thread = row
        regs_up<160>();
        bool ok = true;
        const int r = threadIdx.x - 128;
        const uint32_t lanes = tmem + NS * MB + ((uint32_t)((warp & 3) * 32) << 16);
        float2 acc[D / 2];
        float m = -INFINITY, l = 0.0f; // the softmax's running maximum and sum
        for (int i = 0; i < mine && ok; i++) {
            const ManyTile &x = info[i % INFO];
            if (!(ok = wait(B_INFO_FULL + i % INFO, i / INFO) && wait(B_O_FULL + i % Lay::OS, i / Lay::OS)))
                break;
            tc_after();
            const float *hand = ring + (i % RING) * 3 * MB;
            const float top = hand[r], back = hand[MB + r], sum = hand[2 * MB + r];
            if (x.first) {
                m = -INFINITY;
                l = 0.0f;
            }
            const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.0f : mn;
            const float corr = ex2(m - ref), tile = ex2(top - ref), oscale = tile * back; // 0 from -inf
            l = l * corr + sum * tile;
            m = mn;
            if (x.first) {
#pragma unroll
                for (int d = 0; d < D / 2; d++)
                    acc[d] = make_float2(0.0f, 0.0f);
            }
            const float2 corr2 = make_float2(corr, corr), scale2 = make_float2(oscale, oscale);
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                uint32_t o[16];
                tm_ld16(lanes + (uint32_t)(i % Lay::OS) * D + 16 * k, o);
                tm_wait(o);
                if (k == D / 16 - 1) {
                    tc_before();
                    mbar_arrive(&bar[B_O_EMPTY + i % Lay::OS]);
                }
#pragma unroll
                for (int d = 0; d < 8; d++)
                    acc[8 * k + d] = fma2(acc[8 * k + d], corr2,
                                          mul2(make_float2(__uint_as_float(o[2 * d]), __uint_as_float(o[2 * d + 1])), scale2));
            }
            if (x.last) {
                const int row = x.mt * R + r / rep, head = x.g * rep + r % rep;
                const bool done = x.from_start && x.to_end, live = r < R * rep && row < x.n;
                if (!done && x.from_start && r == 0) {
                    JoinHead h{};
                    h.pieces = x.pieces;
                    h.first = x.mt * R * rep;
                    h.vectors = min(R, x.n - x.mt * R) * rep;
                    h.g = x.g;
                    h.r0 = x.r0;
                    p.head[slot] = h;
                }
                if (live) {
                    const float inv = !done ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
                    T *out = reinterpret_cast<T *>(a.out) + (size_t)(x.r0 + row) * a.ld_out + (size_t)head * D;
                    float *part = p.part + ((size_t)slot * 2 + (x.from_start ? 1 : 0)) * MB * (D + 2);
#pragma unroll
                    for (int d = 0; d < D; d += 16) {
                        float o[16];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            o[2 * j] = acc[d / 2 + j].x * inv;
                            o[2 * j + 1] = acc[d / 2 + j].y * inv;
                        }
                        if (done)
                            store_row<16>(out + d, o);
                        else
                            store_row<16>(part + (size_t)r * D + d, o);
                    }
                    if (!done) {
                        part[(size_t)MB * D + r] = m;
                        part[(size_t)MB * (D + 1) + r] = l;
                    }
                }
            }
            __syncwarp();
            if (lane == 0)
                mbar_arrive(&bar[B_INFO_EMPTY + i % INFO]);
        }
        leave(ok);
    } else if (wg == 2 || wg == 5) {
        // ================================================= codes to f16: keys, values
        regs_down<56>();
        bool ok = true;
        // Eight lanes take eight 16-code units: for D = 128 half the units of two tokens,
        // crosswise, for D = 64 two tokens, so that the eight 16-byte stores of a pass fall
        // into eight bank groups.  Unit n of a thread: token tok + 32 * (n / PER), column
        // unit0 or unit1.
        constexpr int PER = D / 64;      // units of a token pair row that a thread takes
        constexpr int N = 4 * PER;       // units a thread widens per tile
        const bool v = wg == 5;
        const int t = threadIdx.x & 127, j = t & 7, odd = j >> 2;
        const int tok = 2 * (t >> 3) + odd;
        const int unit0 = D == 128 ? 4 * odd + (j & 3) : j & 3, unit1 = unit0 ^ 4;
        const int sw = tok & 7;          // the same for every token of the thread
        auto place = [&](int unit) { return (unit >> 2) * (MB * 128) + tok * 128 + (((2 * (unit & 3)) ^ sw) << 4); };
        const int at0 = place(unit0), at1 = place(unit1);
        uint4 codes[N];
        const int8_t *pool = (v ? a.c.vq : a.c.kq) + (tok & 15) * D + unit0 * 16;
        auto load = [&](int i) { // the thread's units of tile i
            const int *rows = info[i % INFO].row + (tok >> 4);
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const int row = rows[2 * n];
                const int8_t *src = pool + (size_t)row * D;
#pragma unroll
                for (int u = 0; u < PER; u++)
                    codes[n * PER + u] = row >= 0 ? __ldg(reinterpret_cast<const uint4 *>(src + (u ? (unit1 - unit0) * 16 : 0)))
                                                  : make_uint4(0, 0, 0, 0);
            }
            __syncwarp();
            if (lane == 0) // the rows are read
                mbar_arrive(&bar[B_INFO_EMPTY + i % INFO]);
        };
        if ((ok = wait(B_INFO_FULL, 0)))
            load(0);
#pragma unroll 1
        for (int i = 0; i < mine && ok; i++) {
            const int b = i % Lay::KVS, use = i / Lay::KVS;
            if (!(ok = use == 0 || wait((v ? B_V_EMPTY : B_K_EMPTY) + b, use - 1)))
                break;
            uint8_t *dst = smem + (v ? Lay::v_off : Lay::k_off) + b * Lay::T;
#pragma unroll
            for (int n = 0; n < N; n++) {
                uint4 a0, a1;
                widen(codes[n], a0, a1);
                const int at = (n % PER ? at1 : at0) + (n / PER) * 32 * 128;
                *reinterpret_cast<uint4 *>(dst + at) = a0;
                *reinterpret_cast<uint4 *>(dst + (at ^ 16)) = a1;
            }
            fence_proxy_async_smem();
            mbar_arrive(&bar[(v ? B_V_FULL : B_K_FULL) + b]);
            if (i + 1 < mine) {
                if (!(ok = wait(B_INFO_FULL + (i + 1) % INFO, (i + 1) / INFO)))
                    break;
                load(i + 1);
            }
        }
        leave(ok);
    } else if (wg == 3) {
        regs_down<48>();
        bool ok = true;
        if (warp == 12) {
            // ============================================= the products
            constexpr uint32_t QK = idesc_f16(MB, false), PV = idesc_f16(D, true);
            const uint32_t sq = sw128(smem_addr(smem), 16), sk = sw128(smem_addr(smem + Lay::k_off), 16),
                           sv = sw128(smem_addr(smem + Lay::v_off), MB * 128);
            int item = -1;
            auto test = [&](int b, int use) { return __all_sync(0xffffffffu, mbar_test(&bar[b], (uint32_t)(use & 1))); };
            auto qk = [&](int i, bool first, bool last) {
                const int b = i % Lay::KVS;
                // S lies under the P of tile i - NS, which that tile's product has read
                if (!((!first || test(B_Q_FULL + item % Lay::QS, item / Lay::QS)) && test(B_K_FULL + b, i / Lay::KVS) &&
                      (i < NS || test(B_P_EMPTY + i % NS, i / NS - 1))))
                    return false;
                tc_after();
#pragma unroll
                for (int c = QP - 1; c >= 0; c--) // the small pieces first: the accumulator cuts off at every step
#pragma unroll
                    for (int k = 0; k < D / 64; k++)
                        mma_ss4(tmem + (uint32_t)(i % NS) * MB, sq + ((item % Lay::QS * QP + c) * Lay::T + k * MB * 128) / 16,
                                sk + (b * Lay::T + k * MB * 128) / 16, QK, c < QP - 1 || k);
                tc_commit(&bar[B_K_EMPTY + b]);
                if (last)
                    tc_commit(&bar[B_Q_EMPTY + item % Lay::QS]);
                tc_commit(&bar[B_S_FULL + i % NS]);
                return true;
            };
            auto pv = [&](int i) {
                const int b = i % Lay::KVS;
                if (!(test(B_P_FULL + i % NS, i / NS) && test(B_V_FULL + b, i / Lay::KVS) &&
                      (i < Lay::OS || test(B_O_EMPTY + i % Lay::OS, i / Lay::OS - 1))))
                    return false;
                tc_after();
#pragma unroll
                for (int c = PP - 1; c >= 0; c--)
#pragma unroll
                    for (int k = 0; k < 2; k++) // 64 tokens
                        mma_ts4(tmem + NS * MB + (uint32_t)(i % Lay::OS) * D, tmem + (uint32_t)(i % NS) * MB + 64 * k + 8 * c,
                                sv + (b * Lay::T + k * 64 * 128) / 16, PV, c < PP - 1 || k);
                tc_commit(&bar[B_V_EMPTY + b]);
                tc_commit(&bar[B_P_EMPTY + i % NS]);
                tc_commit(&bar[B_O_FULL + i % Lay::OS]);
                return true;
            };
            // whichever is ready: the scores of tile iq, the output of tile ip
            int iq = 0, ip = 0;
            bool known = false, first = false, last = false;
            uint32_t left = 1u << 22; // polls without either
#pragma unroll 1
            while (ip < mine && ok) {
                bool did = false;
                if (iq < mine) {
                    if (!known && test(B_INFO_FULL + iq % INFO, iq / INFO)) {
                        first = __shfl_sync(0xffffffffu, info[iq % INFO].first, 0);
                        last = __shfl_sync(0xffffffffu, info[iq % INFO].last, 0);
                        if (lane == 0)
                            mbar_arrive(&bar[B_INFO_EMPTY + iq % INFO]);
                        item += first;
                        known = true;
                    }
                    if (known && qk(iq, first, last)) {
                        iq++;
                        known = false;
                        did = true;
                    }
                }
                if (ip < iq && pv(ip)) {
                    ip++;
                    did = true;
                }
                if (did)
                    left = 1u << 22;
                else if (--left == 0) {
                    atomicCAS(a.err, 0u, (uint32_t)DEV_ERR_MBAR_TIMEOUT);
                    ok = false;
                } else {
                    __nanosleep(20);
                }
            }
            // every arrival lands before the barriers go
            const int b = (mine - 1) % Lay::KVS, use = (mine - 1) / Lay::KVS;
            ok = ok && wait(B_K_EMPTY + b, use) && wait(B_V_EMPTY + b, use) && wait(B_Q_EMPTY + item % Lay::QS, item / Lay::QS) &&
                 wait(B_P_EMPTY + (mine - 1) % NS, (mine - 1) / NS);
        } else if (warp == 13) {
            // ============================================= pages and scales, ahead
            // Four tiles at a time, eight lanes each: a tile's page and then its scales are two
            // trips to memory, 2000 cycles, and alone a tile would wait for both.
            Walk at;
            int tile = at.start(p, s_seq, s_at, R), item = 0;
            bool from_start = tile == 0;
            const int q = lane >> 3, group = lane & 7;
            for (int i0 = 0; i0 < mine && ok; i0 += 4) {
                Walk own = at; // of tile i0 + q
                int own_tile = tile, own_item = item;
                bool own_start = from_start;
                for (int c = 0; c < 4 && i0 + c < mine; c++) {
                    if (c == q) {
                        own = at;
                        own_tile = tile;
                        own_item = item;
                        own_start = from_start;
                    }
                    if (++tile == at.nt && i0 + c + 1 < mine) {
                        tile = 0;
                        item++;
                        from_start = true;
                        at.next(p, rep, R);
                    }
                }
                const int pos = own_tile * MB + group * 16, need = own.len + min(own.n, (own.mt + 1) * R);
                int row = -1;
                float ks = 0.0f, vs = 0.0f;
                if (pos < need && i0 + q < mine) {
                    const int id = kv8_page(a.b, a.c, own.s, pos / a.c.page, a.err);
                    if (id >= 0) {
                        const size_t o = (size_t)id * a.c.n_kv + own.g;
                        row = (int)(o * a.c.page) + pos % a.c.page;
                        ks = a.c.ks[o];
                        vs = a.c.vs[o];
                    }
                }
                const float lvs = ceilf(log2f(vs));
                const bool hole = (__ballot_sync(0xffffffffu, row < 0) >> (8 * q)) & 255u;
                for (int c = 0; c < 4 && i0 + c < mine && ok; c++) {
                    const int i = i0 + c;
                    if (i >= INFO && !(ok = wait(B_INFO_EMPTY + i % INFO, i / INFO - 1)))
                        break;
                    ManyTile &x = info[i % INFO];
                    if (q == c) {
                        x.row[group] = row;
                        x.ks[group] = ks;
                        x.vs[group] = vs;
                        x.lvs[group] = lvs;
                        if (group == 0) {
                            x.first = i == 0 || own_tile == 0;
                            x.to_end = own_tile == own.nt - 1;
                            x.last = x.to_end || i == mine - 1;
                            x.masked = hole || own_tile * MB + MB > own.len + own.mt * R + 1;
                            x.tile = own_tile;
                            x.g = own.g;
                            x.mt = own.mt;
                            x.r0 = own.r0;
                            x.n = own.n;
                            x.len = own.len;
                            x.from_start = own_start;
                            x.item = own_item;
                            x.pieces = (int)(((lo + i + (own.nt - 1 - own_tile) + 1) * active - 1) / total) - slot + 1;
                        }
                    }
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive(&bar[B_INFO_FULL + i % INFO]);
                }
            }
        } else if (warp == 14) {
            // ============================================= Q of the next rows
            Walk at;
            int begun = at.start(p, s_seq, s_at, R), left = mine; // tiles of the pair in front of this range; tiles left
            int item = 0;
            for (; left > 0 && ok; item++) {
                if (!(ok = item < Lay::QS || wait(B_Q_EMPTY + item % Lay::QS, item / Lay::QS - 1)))
                    break;
                if (lane == 0) {
                    uint64_t *full = &bar[B_Q_FULL + item % Lay::QS];
                    mbar_arrive_expect_tx(full, QP * D * 2 * R * rep);
                    for (int c = 0; c < QP; c++)
                        for (int d = 0; d < D; d += 64)
                            asm volatile(
                                "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
                                " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                                    smem_addr(smem + (item % Lay::QS * QP + c) * Lay::T + d * MB * 2)),
                                "l"(&p.tq), "r"(d), "r"(at.g * rep), "r"(at.r0 + at.mt * R), "r"(c), "r"(smem_addr(full))
                                : "memory");
                }
                __syncwarp();
                left -= at.nt - begun;
                begun = 0;
                if (left > 0)
                    at.next(p, rep, R);
            }
            // copies in flight land before the shared memory goes
            for (int i = max(0, item - Lay::QS); i < item; i++)
                for (int it = 0; it < 100000 && !mbar_try_wait(&bar[B_Q_FULL + i % Lay::QS], (uint32_t)((i / Lay::QS) & 1)); it++)
                    ;
        }
        leave(ok);
        if (warp == 12)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(512) : "memory");
    }
}

// Q of the sequences with many rows, once: rotated by its position, brought to
// [1, 2) by a power of two of each vector's own (f16 holds it whatever its
// magnitude), in QP f16 pieces.  A CTA a row.  Bound by its bytes; inside the
// attention kernel two or four warps took 5 to 25 us for a tile's vectors,
// which the tiles of a prompt's first rows, with few tokens each, waited for.
template <class T, int D, int QP>
__global__ void __launch_bounds__(QT) kv8_q_kernel(const __grid_constant__ ManyParams p)
{
    constexpr int L = D / 8; // lanes of a vector: four dims of each half
    constexpr int H = D / 2;
    const Kv8Attn &a = p.a;
    const int row = blockIdx.x, j = threadIdx.x % L;
    // the row's sequence: the first with many rows, this one among them, whose numbers fit (as
    // kv8_many_kernel judges them, each by its own: the row starts of a bad batch can fall)
    __shared__ int s_owner;
    if (threadIdx.x == 0)
        s_owner = INT_MAX;
    __syncthreads();
    int r0, n, len;
    for (int s = threadIdx.x; s < a.b.n_seqs; s += QT)
        if (a.b.row_start[s] <= row && row < a.b.row_start[s + 1]) {
            kv8_seq(a.b, s, a.err, r0, n, len);
            if ((long long)n * (a.n_heads / a.c.n_kv) > p.many)
                atomicMin(&s_owner, s);
        }
    __syncthreads();
    const int s = s_owner;
    if (s == INT_MAX)
        return;
    kv8_seq(a.b, s, a.err, r0, n, len);
    if (row < r0 || row >= r0 + n) // only if the batch's numbers changed under way
        return;
    const T *q = reinterpret_cast<const T *>(a.q) + (size_t)row * a.ld_q;
    float4 c = make_float4(1.0f, 1.0f, 1.0f, 1.0f), t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (a.r.cos) {
        const size_t o = (size_t)(len + row - r0) * H + 4 * j;
        c = kv8_load4(a.r.cos + o);
        t = kv8_load4(a.r.sin + o);
    }
    for (int h0 = 0; h0 < a.n_heads; h0 += QT / L) { // whole warps: the shuffles are among all lanes
        const int h = h0 + (int)threadIdx.x / L;
        const bool live = h < a.n_heads;
        float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = u;
        if (live) {
            u = kv8_load4(q + (size_t)h * D + 4 * j);
            v = kv8_load4(q + (size_t)h * D + H + 4 * j);
            if (a.r.cos) {
                const float4 w = u;
                u.x = __fsub_rn(__fmul_rn(w.x, c.x), __fmul_rn(v.x, t.x));
                u.y = __fsub_rn(__fmul_rn(w.y, c.y), __fmul_rn(v.y, t.y));
                u.z = __fsub_rn(__fmul_rn(w.z, c.z), __fmul_rn(v.z, t.z));
                u.w = __fsub_rn(__fmul_rn(w.w, c.w), __fmul_rn(v.w, t.w));
                v.x = __fadd_rn(__fmul_rn(w.x, t.x), __fmul_rn(v.x, c.x));
                v.y = __fadd_rn(__fmul_rn(w.y, t.y), __fmul_rn(v.y, c.y));
                v.z = __fadd_rn(__fmul_rn(w.z, t.z), __fmul_rn(v.z, c.z));
                v.w = __fadd_rn(__fmul_rn(w.w, t.w), __fmul_rn(v.w, c.w));
            }
        }
        float big = fmaxf(fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(u.z), fabsf(u.w))),
                          fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
#pragma unroll
        for (int o = 1; o < L; o <<= 1)
            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        int e = (int)((__float_as_uint(big) >> 23) & 255u) - 127;
        e = max(-126, min(126, e));
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        if (!live)
            continue;
        const size_t vec = (size_t)row * a.n_heads + h;
        if (j == 0)
            p.facs[vec] = __uint_as_float((uint32_t)(127 + e) << 23) * a.scale * 1.4426950408889634f;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const float x[4] = {(k ? v.x : u.x) * down, (k ? v.y : u.y) * down, (k ? v.z : u.z) * down,
                                (k ? v.w : u.w) * down};
            __half *o = p.q16 + vec * D + k * H + 4 * j;
            const uint32_t w0 = pack16(x[0], x[1]), w1 = pack16(x[2], x[3]);
            *reinterpret_cast<uint2 *>(o) = make_uint2(w0, w1);
            if constexpr (QP == 2) {
                const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&w0));
                const float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&w1));
                *reinterpret_cast<uint2 *>(o + (size_t)a.b.n_rows * a.n_heads * D) =
                    make_uint2(pack16(x[0] - f0.x, x[1] - f0.y), pack16(x[2] - f1.x, x[3] - f1.y));
            }
        }
    }
}

template <class T, int D, int QP, int PP>
int run(ManyParams &p, int ctas, cudaStream_t stream)
{
    auto fn = tensor_map_encoder();
    if (!fn)
        return fail(LLMRS_ECUDA, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t heads = p.a.n_heads, rows = p.a.b.n_rows;
    const cuuint32_t rep = p.a.n_heads / p.a.c.n_kv;
    const cuuint64_t dims[4] = {D, heads, rows, QP};
    const cuuint64_t strides[3] = {D * 2, heads * D * 2, rows * heads * D * 2};
    const cuuint32_t box[4] = {64, rep, MB / rep, 1}, estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(&p.tq, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, p.q16, dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(LLMRS_ECUDA, "cuTensorMapEncodeTiled (prepared Q) failed (%d)", (int)r);
    LLMRS_CUDA_TRY(launch(kv8_q_kernel<T, D, QP>, dim3(p.a.b.n_rows), dim3(QT), 0, stream, false, p));
    LLMRS_CUDA_TRY(launch(kv8_many_kernel<T, D, QP, PP>, dim3(ctas), dim3(MANY_THREADS), ManyLay<D, QP>::bytes, stream,
                          true, p));
    LLMRS_CUDA_TRY(launch(kv8_join_kernel<T, D, MB>, dim3(8 * ctas), dim3(JT), 0, stream, true, p.a,
                          (const float *)p.part, (const JoinHead *)p.head, ctas));
    return LLMRS_OK;
}

template <class T, int D, int QP, int PP>
cudaError_t prepare()
{
    return cudaFuncSetAttribute(kv8_many_kernel<T, D, QP, PP>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                ManyLay<D, QP>::bytes);
}

} // namespace

static size_t pieces_bytes(int head_dim)
{
    const size_t bytes = (size_t)MANY_CTAS * (sizeof(JoinHead) + 2 * (size_t)MB * (head_dim + 2) * sizeof(float));
    return (bytes + 255) & ~(size_t)255;
}

size_t kv8_many_workspace(int head_dim, int n_heads, int n_rows)
{
    return pieces_bytes(head_dim) + (size_t)n_rows * n_heads * (2 * head_dim * sizeof(__half) + sizeof(float));
}

int kv8_many_prepare(void)
{
    cudaError_t e = prepare<float, 128, 2, 2>();
    if (e == cudaSuccess)
        e = prepare<float, 64, 2, 2>();
    if (e == cudaSuccess)
        e = prepare<__half, 128, 2, 2>();
    if (e == cudaSuccess)
        e = prepare<__half, 64, 2, 2>();
    if (e == cudaSuccess)
        e = prepare<__nv_bfloat16, 128, 2, 1>();
    if (e == cudaSuccess)
        e = prepare<__nv_bfloat16, 64, 2, 1>();
    if (e != cudaSuccess)
        return fail(LLMRS_ECUDA, "kv8 kernel attributes: %s", cudaGetErrorString(e));
    return LLMRS_OK;
}

int kv8_many(const Kv8Attn &a, int many, void *ws, int sms, cudaStream_t stream)
{
    ManyParams p{};
    p.a = a;
    p.head = reinterpret_cast<JoinHead *>(ws);
    p.part = reinterpret_cast<float *>(p.head + MANY_CTAS);
    p.q16 = reinterpret_cast<__half *>(reinterpret_cast<uint8_t *>(ws) + pieces_bytes(a.c.D));
    p.facs = reinterpret_cast<float *>(p.q16 + 2 * (size_t)a.b.n_rows * a.n_heads * a.c.D);
    p.many = many;
    const int ctas = sms < MANY_CTAS ? sms : MANY_CTAS;
    if (a.dtype == LLMRS_F32)
        return a.c.D == 128 ? run<float, 128, 2, 2>(p, ctas, stream) : run<float, 64, 2, 2>(p, ctas, stream);
    if (a.dtype == LLMRS_F16)
        return a.c.D == 128 ? run<__half, 128, 2, 2>(p, ctas, stream) : run<__half, 64, 2, 2>(p, ctas, stream);
    return a.c.D == 128 ? run<__nv_bfloat16, 128, 2, 1>(p, ctas, stream)
                        : run<__nv_bfloat16, 64, 2, 1>(p, ctas, stream);
}

} // namespace llmrs
