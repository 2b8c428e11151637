// Attention and its backward, which recomputes the probabilities from the saved log-sum-exp.
#include <math.h>

#include "om_common.cuh"
#include "om_f2.cuh"
#include "om_tc_ptx.cuh"

namespace omb {
namespace attn {

using namespace omb::tc;

// Division of 0 <= n < 2^31 by a divisor known on the host: n * mul / 2^(32 + shift)
// (Granlund and Montgomery, 1994)
struct Div {
    uint32_t d, mul, shift;
    __device__ __forceinline__ int operator()(int n) const {
        return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift);
    }
};
static Div div_by(uint32_t d) {
    Div r = {d, 0, 0};
    if (d <= 1) return r;
    int l = 0;
    while ((1ull << l) < d) ++l;              // 2^(l-1) < d <= 2^l
    r.shift = l - 1;                          // mul = ceil(2^(31 + l) / d) < 2^32
    r.mul = (uint32_t)(((1ull << (31 + l)) + d - 1) / d);
    return r;
}
struct View {          // a [batch, token, head, D] tensor: element strides, D contiguous
    void* p;
    long long sb, st, sh;
};
struct Params {
    View q, k, v, o, dout, dq, dk, dv;
    float* lse;        // [B, H, Sq]
    uint8_t* stat;     // the backward's workspace: see stat_tile
    float2* qmax;      // ... and, for fp16, what bounds the score gradients: see range_factor
    float* vmax;
    const int *qlens, *kvlens;
    int B, H, Hkv, Sq, Sk, D, causal;
    float scale;
    float inv_scale;   // 1 / |scale|, for the backward
    float scale2;      // |scale| * log2(e), not 0 (masked scores stay minus infinity)
    bool neg;          // scale < 0: the score products negate Q
    unsigned int* err;
    int items;         // the forward's tiles times parts, and the divisions that find an item's place
    Div by_splits, by_fast, by_heads;   // by_fast: tiles of a head, causal: heads
    int splits;        // parts of the streamed axis, each CTA one of them (1: no partial results)
    float* part;       // partial results: fp32 rows [split][batch][head][token][D]
    float* part_lse;   // forward: the parts' log2(sum exp) [split][batch][head][token]
};

template <int DT>
__device__ __forceinline__ const typename Half16<DT>::T* row(const View& v, int b, int t, int h) {
    return static_cast<const typename Half16<DT>::T*>(v.p) + b * v.sb + t * v.st + h * v.sh;
}
template <int DT>
__device__ __forceinline__ typename Half16<DT>::T* row_out(const View& v, int b, int t, int h) {
    return static_cast<typename Half16<DT>::T*>(v.p) + b * v.sb + t * v.st + h * v.sh;
}
__device__ __forceinline__ int len_of(const int* lens, int b, int most) {
    return lens ? min(max(lens[b], 0), most) : most;
}
// ---------------------------------------------------------------- tcgen05 pieces
// The low word of a shared-memory descriptor moves with the operand's address; the high word
// (8 rows of 128 bytes apart, 128-byte swizzle) is the same for every operand here. The products
// are issued by one thread, so each takes few instructions: the descriptors of a tile's steps are
// its first one plus constants.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (LAYOUT_SW128 << 29);
// The whole warp runs the issuing code, so that addresses stay in uniform registers (under a
// branch on one lane each product cost about 85 clocks of register moves); `leader` is 1 in the one
// lane whose instruction takes effect.
template <bool ACC>
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .b64 a, b;\n\t.reg .pred p, q;\n\t"
        "mov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(DESC_HI), "n"(ACC ? 1 : 0), "r"(leader));
}
// D[tmem] (+)= A[tmem] * B[smem]: A holds 16-bit pairs, one row per lane, K along the columns.
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo,
                                       uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .b64 b;\n\t.reg .pred p, q;\n\t"
        "mov.b64 b, {%2, %4};\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(DESC_HI), "r"(accumulate), "r"(leader));
}
__device__ __forceinline__ void commit(uint32_t leader, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ uint32_t elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(one));
    return one;
}
// a value that is the same in every lane, in a uniform register (the warp reduction writes one)
__device__ __forceinline__ int uniform(int v) { return __reduce_max_sync(~0u, v); }
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __reduce_max_sync(~0u, v); }
// one arrival for the whole warp, behind what its lanes have done
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if (threadIdx.x % 32 == 0) mbar_arrive(bar);
}
// a bounded wait of a whole warp
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    return __all_sync(~0u, mbar_wait(bar, parity, abort_flag));
}
// 32 columns of this warp's lanes, without waiting: tmem_ld_wait orders the registers.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
          "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
          "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
          "=r"(v[31])
        : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_ld_wait(uint32_t* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(v[i]));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
        "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
        "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]),
        "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
        "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <int DT>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    const auto v = Half16<DT>::pack(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Instruction descriptor of kind::f16 with an fp32 accumulator and M = 128; b_mn: B is stored
// with N contiguous; neg_a: A is negated.
__device__ __forceinline__ uint32_t idesc_f16(bool f16, int n, bool b_mn, bool neg_a) {
    const uint32_t fmt = f16 ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)neg_a << 13) |
           ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// A [128 rows, DP] 16-bit tile lies in shared memory as DP / 64 panels of 128 rows x 128 bytes
// with the 128-byte swizzle, as TMA writes it.
constexpr int PANEL = 128 * 128;
// Low descriptor words. K-major operand (rows = M or N, K = the head dimension): 16 columns are 32
// bytes, 64 a panel. MN-major operand (rows = K, N = the head dimension): 16 rows are 2048 bytes,
// panels of 64 columns as far apart as they are long.
__device__ __forceinline__ uint32_t desc_k(uint32_t tile) { return (tile >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn(uint32_t tile, int panel) { return (tile >> 4) | ((uint32_t)(panel >> 4) << 16); }
// D (+)= X Y^T over the head dimension, ks steps of 16 (X: a tile of 128 rows, Y: of ROWS)
template <int DP, int ROWS, bool ACC = false>
__device__ __forceinline__ void product_k(uint32_t leader, uint32_t d_tmem, uint32_t x, uint32_t y, uint32_t idesc, int ks) {
    const uint32_t a = desc_k(x), b = desc_k(y);
    mma_ss<ACC>(leader, d_tmem, a, b, idesc);
#pragma unroll
    for (int k = 1; k < DP / 16; ++k)
        if (k < ks)
            mma_ss<true>(leader, d_tmem, a + (k / 4) * (PANEL >> 4) + (k % 4) * 2,
                         b + (k / 4) * (ROWS * 128 >> 4) + (k % 4) * 2, idesc);
}
// D (+)= A Y over Y's ROWS rows; columns CW w .. of A are the CW / 2 words at a_tmem + CW w
template <int CW, int ROWS>
__device__ __forceinline__ void product_mn(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t y, uint32_t idesc, bool accumulate) {
    const uint32_t b = desc_mn(y, ROWS * 128);
    mma_ts(leader, d_tmem, a_tmem, b, idesc, accumulate);
#pragma unroll
    for (int k = 1; k < ROWS / 16; ++k)
        mma_ts(leader, d_tmem, a_tmem + k * 16 / CW * CW + k * 16 % CW / 2, b + k * 128, idesc, 1);
}
template <int DP, int ROWS = 128>
__device__ __forceinline__ void load_tile(uint32_t dst_off, uint8_t* smem, const CUtensorMap* map,
                                          uint64_t* bar, int t0, int h, int b) {
#pragma unroll
    for (int c = 0; c < DP / 64; ++c)
        tma_load_4d(smem + dst_off + c * ROWS * 128, map, bar, c * 64, t0, h, b);
}
// Rows [first, ROWS) of a tile become zeros: what lies past a sequence's length must not reach a
// product, since 0 * NaN is NaN. One thread per row.
template <int DP, int ROWS = 128>
__device__ __forceinline__ void zero_tail(uint8_t* tile, int first, int row) {
    if (row >= first && row < ROWS) {
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                reinterpret_cast<uint4*>(tile + c * ROWS * 128 + row * 128)[i] = make_uint4(0, 0, 0, 0);
    }
    fence_async_smem();
}

// Columns c .. c + 31 of row `row` from the accumulators o (zeros unless `any`), times f: rounded into
// the 128-row tile at `tile` (panels of 64 columns with the 128-byte swizzle, for a TMA store: stored
// from the registers, 16 bytes to each of 32 rows at a time, the epilogue took 2400 to 4200 clocks of
// a CTA), or in fp32 to a row of partial results, when it is there.
template <int DT>
__device__ __forceinline__ void store_chunk(const uint32_t (&o)[32], bool any, float f, bool partial, uint8_t* tile, int row,
                                            float* part, int c, int D) {
    const int n8 = min(32, D - c) / 8;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        float v[8];
#pragma unroll
        for (int y = 0; y < 8; ++y) v[y] = any ? __uint_as_float(o[x * 8 + y]) * f : 0.f;
        if (!partial) {
            *reinterpret_cast<uint4*>(tile + c / 64 * PANEL + row * 128 + (((c % 64 / 8 + x) ^ (row & 7)) << 4)) =
                make_uint4(pack16<DT>(v[0], v[1]), pack16<DT>(v[2], v[3]), pack16<DT>(v[4], v[5]), pack16<DT>(v[6], v[7]));
        } else if (part && x < n8) {
            reinterpret_cast<float4*>(part + c)[2 * x] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(part + c)[2 * x + 1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
}
// A tile's panels to rows t0 .. of one batch entry and head; what lies past the tensor is dropped.
__device__ __forceinline__ void store_tile(const CUtensorMap* map, const uint8_t* tile, int D, int t0, int h, int b) {
    for (int c = 0; c < D; c += 64)
        asm volatile(
            "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                reinterpret_cast<uint64_t>(map)), "r"(smem_u32(tile + c / 64 * PANEL)), "r"(c), "r"(t0), "r"(h), "r"(b)
            : "memory");
}
constexpr float LN2 = 0.6931471805599453f;

// ---------------------------------------------------------------- forward
// One item of work: NT tiles of 128 queries of one (batch, head) over the blocks of KB keys (or one
// part of them). A CTA stays on its SM and takes every gridDim.x-th item: a softmax warpgroup per
// tile (thread = query row), a TMA warp and an MMA warp, each running ahead of the others as far as
// the buffers go, so that an item's loads and first scores come beside the last one's end (with a
// CTA per item the time between two CTAs of an SM, about 2.9 us with their set-up, was a third of
// the 54 us that 768 heads of 197 tokens took).
// Per tile and block:
//   S = Q K^T (TMEM, fp32) -> running maximum, P = exp(S - m), row sums -> P (TMEM, 16-bit, over
//   S's columns) -> O += P V (TMEM, fp32).
// The running maximum and sum are those of Milakov and Gimelshein (2018). O is rescaled only when a
// row's maximum has grown by more than 2^8 since its last reference maximum (a known refinement): P
// stays below 2^8, in range of both types, and the factor cancels in O / l.
// Score tile n = NT j + t (block j, query tile t) lies in TMEM buffer n % NB, counted over all items.
// There are more buffers than query tiles, so that a tile's next scores are there when its
// probabilities are done (without, a softmax warp waited about 900 of 2900 clocks a block for them):
// blocks of KB = 128 keys and three buffers for two tiles of heads up to 64 (24 heads of 4096 tokens,
// with 168 registers a thread: 154 us, with 64 keys 176 us). Longer heads' O fills half of TMEM, and
// with one tile two CTAs share an SM, so there are two buffers of 64 keys a tile (768 heads of 64
// queries over 2000 keys: 98 us, with one buffer of 128 keys 121 us).
// TMEM: NB score tiles, then the O tiles.
template <int DP, int NT>
struct FwdCfg {
    static constexpr int KB = DP == 128 || NT == 1 ? 64 : 128;
    static constexpr int TILE = DP / 64 * PANEL, KV_TILE = DP / 64 * KB * 128;
    static constexpr int SLOTS = NT == 2 ? (DP == 128 ? 8 : 6) : (DP == 128 ? 4 : 8);
    // the output's staging tiles: Q's with long heads, which shared memory then holds no others beside
    static constexpr bool OWN_STAGE = DP == 64;
    static constexpr int KV_OFF = NT * TILE, STAGE_OFF = OWN_STAGE ? KV_OFF + SLOTS * KV_TILE : 0;
    static constexpr int BAR_OFF = KV_OFF + SLOTS * KV_TILE + (OWN_STAGE ? NT * TILE : 0);
    static constexpr int SMEM = BAR_OFF + 512;
    // A row's 128 scores and what goes with them need more than the 168 registers that 320 or 384
    // threads can have each (114 bytes spilled): the softmax warps take what the other warpgroup,
    // whose last two warps idle, gives back. 24 heads of 4096 tokens: 154 -> 145 us
    static constexpr bool MORE_REGS = KB == 128;
    static constexpr int THREADS = NT * 128 + (MORE_REGS ? 128 : 64), OCC = NT == 1 ? 2 : 1;
    static constexpr int MATH_REGS = 208, OTHER_REGS = 80;
    // Registers a thread that the launch must have for that split, else the softmax warps would wait.
    // The compiler gives such a kernel all that its launch bounds allow (168); the host checks it
    static constexpr int LAUNCH_REGS = MORE_REGS ? (NT * 128 * MATH_REGS + 128 * OTHER_REGS + THREADS - 1) / THREADS : 0;
    static constexpr int TMEM_COLS = NT * 256;
    static constexpr int NB = KB == 64 ? 2 * NT : 3;
    static constexpr int O_COL = NB * KB, O_STEP = DP;
    static_assert(O_COL + NT * O_STEP <= TMEM_COLS && (SMEM + 1024) * OCC <= 228 * 1024, "on-chip memory");
};
enum : unsigned int { ERR_LOAD = ERRBIT_TC_PRODUCER, ERR_MMA = ERRBIT_TC_MMA,
                      ERR_MATH = ERRBIT_TC_EPILOGUE, ERR_DRAIN = ERRBIT_TC_DRAIN };

struct FwdPlace { int b, h, q0, split; };
struct FwdRange { int ql, kl, blk0, nblk; };
// The r-th item of a CTA, in turns from the first and from the last CTA (long items come first), or
// one past the end.
__device__ __forceinline__ int fwd_at(int r) {
    return r * gridDim.x + (r % 2 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}
template <int NT>
__device__ __forceinline__ FwdPlace fwd_place(const Params& p, int at) {
    // causal: heads fastest and the longest rows first, so that the last items are short
    const int i = p.by_splits(at), hi = p.by_fast(i), lo = i - hi * (int)p.by_fast.d;
    const int bh = p.causal ? lo : hi, tile = p.causal ? (p.Sq + NT * 128 - 1) / (NT * 128) - 1 - hi : lo;
    const int b = p.by_heads(bh);
    return {b, bh - b * p.H, tile * (NT * 128), at - i * p.splits};
}
template <int NT, int KB>
__device__ __forceinline__ FwdRange fwd_range(const Params& p, const FwdPlace& w) {
    FwdRange r;
    r.ql = len_of(p.qlens, w.b, p.Sq);
    r.kl = len_of(p.kvlens, w.b, p.Sk);
    int end = w.q0 < r.ql ? r.kl : 0;
    if (p.causal) end = min(end, min(w.q0 + NT * 128, r.ql) + r.kl - r.ql);
    // this part's key blocks: blk0 .. blk0 + nblk - 1
    const int all = end > 0 ? (end + KB - 1) / KB : 0, share = p.by_splits(all + p.splits - 1);
    r.blk0 = w.split * share;
    r.nblk = uniform(max(0, min(all - r.blk0, share)));
    return r;
}

template <int DP, int NT, int DT>
__global__ void __launch_bounds__(FwdCfg<DP, NT>::THREADS, FwdCfg<DP, NT>::OCC)
attn_fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mo, const Params p) {
    using Cf = FwdCfg<DP, NT>;
    // aligned by its declaration, so that every address below is a constant (rounded up at run time,
    // the barriers' pointers took the registers that the scores need)
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) % 1024) {
        if (threadIdx.x == 0) atomicOr(p.err, ERR_LOAD);
        return;
    }
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cf::BAR_OFF);
    // q_full and q_empty pass once an item, with key blocks or without. Only warps that arrive on
    // q_empty wait for q_full, each time: so none is ever two phases of a barrier behind another
    uint64_t *q_full = bars, *q_empty = bars + 1, *drain = bars + 2;
    uint64_t* s_full = bars + 3;                 // per score buffer
    uint64_t* p_full = s_full + Cf::NB;
    uint64_t* pv_done = p_full + Cf::NB;         // per tile: O has a block's product
    uint64_t* o_full = pv_done + NT;             // ... and the item's last one
    uint64_t* o_free = o_full + NT;              // ... and has been read by the item's epilogue
    uint64_t* out_ready = o_free + NT;           // the staging tile is written
    uint64_t* stage_free = out_ready + NT;       // ... and stored
    uint64_t* full = stage_free + NT;
    uint64_t* empty = full + Cf::SLOTS;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(empty + Cf::SLOTS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

    const int warp = uniform((int)threadIdx.x / 32), lane = threadIdx.x % 32;
    constexpr int W_LOAD = NT * 4, W_MMA = NT * 4 + 1, KB = Cf::KB;
    const int items = p.items;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1 + NT);
        mbar_init(drain, 1);
        for (int i = 0; i < Cf::NB; ++i) { mbar_init(s_full + i, 1); mbar_init(p_full + i, 4); }
        for (int t = 0; t < NT; ++t) {
            mbar_init(pv_done + t, 1);
            mbar_init(o_full + t, 1);
            mbar_init(o_free + t, 4);
            mbar_init(out_ready + t, 4);
            mbar_init(stage_free + t, 1);
        }
        for (int i = 0; i < Cf::SLOTS; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_holder)), "r"(Cf::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(*tmem_holder);
    unsigned int err = 0;
    if (Cf::MORE_REGS && warp >= W_LOAD) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cf::OTHER_REGS));

    if (warp == W_LOAD) {
        int slot = 0, issued = 0, queries = 0;   // queries: phases of q_full so far
        uint32_t slot_ph = 1, item_ph = 1;
        bool ok = true;
        for (int turn = 0; ok && turn * (int)gridDim.x < items; ++turn) {
            const int at = fwd_at(turn);
            if (at >= items) continue;
            const FwdPlace w = fwd_place<NT>(p, at);
            const FwdRange r = fwd_range<NT, Cf::KB>(p, w);
            ok = warp_wait(q_empty, item_ph, abort_flag);
            if (!ok) break;
            item_ph ^= 1;
            if (lane == 0 && r.nblk > 0) {
                mbar_expect_tx(q_full, NT * Cf::TILE);
                for (int t = 0; t < NT; ++t) load_tile<DP>(t * Cf::TILE, smem, &mq, q_full, w.q0 + t * 128, w.h, w.b);
            } else if (lane == 0) {
                mbar_arrive(q_full);
            }
            ++queries;
            const int hk = w.h / (p.H / p.Hkv);
            for (int i = 0; i < 2 * r.nblk; ++i) {   // K, V of each block
                ok = warp_wait(empty + slot, slot_ph, abort_flag);
                if (!ok) break;
                if (lane == 0) {
                    mbar_expect_tx(full + slot, Cf::KV_TILE);
                    load_tile<DP, KB>(Cf::KV_OFF + slot * Cf::KV_TILE, smem, i & 1 ? &mv : &mk, full + slot,
                                      (r.blk0 + i / 2) * KB, hk, w.b);
                }
                ++issued;
                if (++slot == Cf::SLOTS) { slot = 0; slot_ph ^= 1; }
            }
        }
        if (!ok || *abort_flag) {                // every load issued has to land before the CTA ends
            *abort_flag = 1;
            err = ok ? 0 : ERR_LOAD;
            if (queries > 0 && !mbar_wait_drain(q_full, (queries - 1) & 1)) err |= ERR_DRAIN;
            for (int j = max(0, issued - Cf::SLOTS); j < issued; ++j)
                if (!mbar_wait_drain(full + j % Cf::SLOTS, (j / Cf::SLOTS) & 1)) err |= ERR_DRAIN;
        }
    } else if (warp == W_MMA) {
        const uint32_t leader = elect();
        const int ks = (p.D + 15) / 16;
        const uint32_t id_s = idesc_f16(DT == OM_DTYPE_F16, KB, false, p.neg);
        const uint32_t id_o = idesc_f16(DT == OM_DTYPE_F16, ks * 16, true, false);
        const uint32_t q_tile = smem_u32(smem), kv_base = q_tile + Cf::KV_OFF;
        // Running places: slot and TMEM buffer of the scores to issue next (sn) and of the
        // probabilities to take next (pn), counted over all items
        struct { int tile, slot, buf; uint32_t slot_ph, buf_ph; } sn = {0, 0, 0, 0, 0}, pn = {0, 1, 0, 0, 0};
        auto step = [&](auto& at) {
            if (++at.buf == Cf::NB) { at.buf = 0; at.buf_ph ^= 1; }
            if (++at.tile == NT) {
                at.tile = 0;
                at.slot += 2;
                if (at.slot >= Cf::SLOTS) { at.slot -= Cf::SLOTS; at.slot_ph ^= 1; }
            }
        };
        auto scores = [&]() {             // one score tile, and K's slot back behind the block's last
            if (sn.tile == 0 && !warp_wait(full + sn.slot, sn.slot_ph, abort_flag)) return false;
            tc_fence_after();
            product_k<DP, KB>(leader, tmem + sn.buf * KB, q_tile + sn.tile * Cf::TILE, kv_base + sn.slot * Cf::KV_TILE,
                               id_s, ks);
            commit(leader, s_full + sn.buf);
            if (sn.tile == NT - 1) commit(leader, empty + sn.slot);
            step(sn);
            return true;
        };
        uint32_t q_ph = 0, o_ph = 1;      // o_ph: the first item finds O free
        bool ok = true;
        for (int turn = 0; ok && turn * (int)gridDim.x < items; ++turn) {
            const int at = fwd_at(turn);
            if (at >= items) continue;
            const FwdRange r = fwd_range<NT, Cf::KB>(p, fwd_place<NT>(p, at));
            const int total = NT * r.nblk;
            ok = warp_wait(q_full, q_ph, abort_flag);
            if (!ok) break;
            q_ph ^= 1;
            if (total == 0) {
                if (leader) mbar_arrive(q_empty);
                continue;
            }
            int issued = 0;
            for (; ok && issued < Cf::NB && issued < total; ++issued) ok = scores();
            if (ok && issued == total) commit(leader, q_empty);
            for (int n = 0; ok && n < total; ++n) {
                const int t = pn.tile;
                ok = (t > 0 || warp_wait(full + pn.slot, pn.slot_ph, abort_flag)) &&
                     (n >= NT || warp_wait(o_free + t, o_ph, abort_flag)) &&
                     warp_wait(p_full + pn.buf, pn.buf_ph, abort_flag);
                if (!ok) break;
                tc_fence_after();
                product_mn<KB, KB>(leader, tmem + Cf::O_COL + t * Cf::O_STEP, tmem + pn.buf * KB,
                                   kv_base + pn.slot * Cf::KV_TILE, id_o, n >= NT);
                commit(leader, pv_done + t);
                if (n >= total - NT) commit(leader, o_full + t);
                if (t == NT - 1) commit(leader, empty + pn.slot);
                step(pn);
                if (issued < total) {     // behind the product that read the buffer's probabilities
                    ok = scores();
                    if (ok && ++issued == total) commit(leader, q_empty);
                }
            }
            o_ph ^= 1;
        }
        if (!ok) {                        // no MMA may run on when the CTA ends
            *abort_flag = 1;
            err = ERR_MMA;
            commit(leader, drain);
            if (!mbar_wait_drain(drain, 0)) err |= ERR_DRAIN;
        }
    } else if (warp < W_LOAD) {
        if (Cf::MORE_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cf::MATH_REGS));
        const int t = warp / 4, row = (warp % 4) * 32 + lane;
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;
        const uint32_t o_addr = tmem + Cf::O_COL + t * Cf::O_STEP + lanes;
        uint8_t* stage = smem + Cf::STAGE_OFF + t * Cf::TILE;
        int buf = t, vslot = 1;           // running places, as the MMA warp's
        uint32_t buf_ph = 0, v_ph = 0, pv_ph = 1, o_ph = 0, out_ph = 0;
        bool ok = true;
        for (int turn = 0; ok && turn * (int)gridDim.x < items; ++turn) {
            const int at = fwd_at(turn);
            if (at >= items) continue;
            int row_end, kl_left, nblk;       // from the part's first key block on
            {
                const FwdPlace w = fwd_place<NT>(p, at);
                const FwdRange r = fwd_range<NT, Cf::KB>(p, w);
                const int i = w.q0 + t * 128 + row;
                row_end = i < r.ql ? r.kl : 0;
                if (p.causal) row_end = min(row_end, i + r.kl - r.ql + 1);
                row_end -= r.blk0 * KB;
                kl_left = r.kl - r.blk0 * KB;
                nblk = r.nblk;
            }
            float m = -INFINITY, l = 0.f;
            // this warpgroup's part in q_empty: here with staging tiles of their own, else at the end
            auto seen_item = [&]() {
                if (Cf::OWN_STAGE && warp % 4 == 0) {
                    if (lane == 0) mbar_arrive(q_empty);
                    __syncwarp();
                }
            };
            if (nblk == 0 && warp % 4 == 0) {
                ok = warp_wait(q_full, out_ph, abort_flag);
                if (!ok) break;
                seen_item();
            }
            for (int j = 0; j < nblk; ++j) {
                const uint32_t s_addr = tmem + buf * KB + lanes;
                ok = warp_wait(s_full + buf, buf_ph, abort_flag);
                if (!ok) break;
                if (j == 0) seen_item();
                tc_fence_after();
                const int seen = row_end - j * KB;              // columns of this block that the row sees
                uint32_t sv[KB];
#pragma unroll
                for (int c = 0; c < KB / 32; ++c) tmem_ld32_issue(s_addr + c * 32, sv + c * 32);
                tmem_ld_wait<KB>(sv);
                float* s = reinterpret_cast<float*>(sv);
                if (__any_sync(~0u, seen < KB)) {
#pragma unroll
                    for (int c = 0; c < KB; ++c) s[c] = c < seen ? s[c] : -INFINITY;
                }
                float mx[4] = {m, s[0], s[1], s[2]};
#pragma unroll
                for (int c = 3; c < KB - 1; c += 2) mx[c / 2 % 4] = max3(mx[c / 2 % 4], s[c], s[c + 1]);
                const float m_new = max3(fmaxf(mx[0], s[KB - 1]), mx[1], fmaxf(mx[2], mx[3]));
                // the reference maximum moves when a row's maximum has grown by more than 2^8
                const bool grow = j > 0 && __any_sync(~0u, (m_new - m) * p.scale2 > 8.f);
                float f = 1.f;
                if (j == 0) {
                    m = m_new;
                } else if (grow) {
                    f = m == -INFINITY ? 0.f : ex2((m - m_new) * p.scale2);
                    l *= f;
                    m = m_new;
                }
                const float sub = m == -INFINITY ? 0.f : -m * p.scale2;
                const F2 sc = {p.scale2, p.scale2}, sb = {sub, sub};
                F2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
                for (int c = 0; c < KB / 32; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        F2 e = fma2({s[c * 32 + 2 * x], s[c * 32 + 2 * x + 1]}, sc, sb);
                        e.x = ex2(e.x);
                        e.y = ex2(e.y);
                        sum[x % 2] = add2(sum[x % 2], e);
                        w[x] = pack16<DT>(e.x, e.y);
                    }
                    tmem_st16(s_addr + c * 16, w);
                }
                sum[0] = add2(sum[0], sum[1]);
                l += sum[0].x + sum[0].y;
                // behind the last product that added to O; the one before that was complete before S of
                // this block was, so the phase is told by its parity
                if (grow) {
                    ok = warp_wait(pv_done + t, pv_ph, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    for (int c = 0; c < p.D; c += 32) {
                        uint32_t o[32];
                        tmem_ld32_issue(o_addr + c, o);
                        tmem_ld_wait<32>(o);
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                        tmem_st32(o_addr + c, o);
                    }
                }
                // keys past the sequence's length may hold anything
                if (t == 0 && kl_left - j * KB < KB) {
                    ok = warp_wait(full + vslot, v_ph, abort_flag);
                    if (!ok) break;
                    zero_tail<DP, KB>(smem + Cf::KV_OFF + vslot * Cf::KV_TILE, kl_left - j * KB, row);
                }
                tmem_st_wait();
                tc_fence_before();
                warp_arrive(p_full + buf);
                buf += NT;
                if (buf >= Cf::NB) { buf -= Cf::NB; buf_ph ^= 1; }
                vslot += 2;
                if (vslot >= Cf::SLOTS) { vslot -= Cf::SLOTS; v_ph ^= 1; }
                pv_ph ^= 1;               // the phase of this block's product, the next block's last one
            }
            // o_full passes once an item and is waited for each time; pv_done's last phase must not
            // be waited for here, since the one before it may still be open
            if (ok && nblk > 0) {
                ok = warp_wait(o_full + t, o_ph, abort_flag);
                o_ph ^= 1;
            }
            // the last item's output has left the staging tile
            if (ok && p.splits == 1) ok = warp_wait(stage_free + t, out_ph ^ 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            int again = at;               // worked out again rather than held through the blocks
            asm volatile("" : "+r"(again));
            const FwdPlace w = fwd_place<NT>(p, again);
            const int i = w.q0 + t * 128 + row;
            const float inv = l == 0.f ? 0.f : 1.f / l;    // 0: no key seen; NaN stays NaN, also in lse
            const long long rows = (long long)p.B * p.H * p.Sq, to = ((long long)w.b * p.H + w.h) * p.Sq + i;
            float* part = i < p.Sq && p.splits > 1 ? p.part + (w.split * rows + to) * p.D : nullptr;
            for (int c = 0; c < p.D; c += 32) {
                uint32_t o[32];
                if (nblk > 0) {
                    tmem_ld32_issue(o_addr + c, o);
                    tmem_ld_wait<32>(o);
                }
                store_chunk<DT>(o, nblk > 0, inv, p.splits > 1, stage, row, part, c, p.D);
            }
            if (nblk > 0) {
                tc_fence_before();
                warp_arrive(o_free + t);
            }
            if (i < p.Sq) {
                // l is relative to the rounded product, as `sub` had it: fused with the sum, it would not be
                const float lse2 = l == 0.f ? -INFINITY : __fadd_rn(__fmul_rn(m, p.scale2), log2f(l));
                if (p.splits > 1)
                    p.part_lse[w.split * rows + to] = lse2;
                else if (p.lse)
                    p.lse[to] = lse2 * LN2;
            }
            if (p.splits == 1) {
                fence_async_smem();
                warp_arrive(out_ready + t);
                if (warp % 4 == 0) {
                    ok = warp_wait(out_ready + t, out_ph, abort_flag);
                    if (!ok) break;
                    if (lane == 0) {
                        if (w.q0 + t * 128 < p.Sq) {
                            store_tile(&mo, stage, p.D, w.q0 + t * 128, w.h, w.b);
                            bulk_commit();
                            bulk_wait_read<0>();
                        }
                        mbar_arrive(stage_free + t);
                        if (!Cf::OWN_STAGE) mbar_arrive(q_empty);
                    }
                    __syncwarp();
                }
            } else if (!Cf::OWN_STAGE) {
                if (warp % 4 == 0 && lane == 0) mbar_arrive(q_empty);
                __syncwarp();
            }
            out_ph ^= 1;
        }
        if (!ok) {
            *abort_flag = 1;
            err = ERR_MATH;
        }
    }
    if (err) atomicOr(p.err, err);
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cf::TMEM_COLS));
    }
}

// ---------------------------------------------------------------- backward
// Both backward kernels are one template. KV = false (dQ): a CTA keeps Q and dO of 128 queries
// and streams key/value blocks; KV = true (dK, dV): it keeps K and V of 128 keys and streams Q
// and dO blocks of every query head that shares them. With X1, X2 the kept tiles and Y1, Y2 the
// streamed ones, per block:
//   S = X1 Y1^T, dP = X2 Y2^T                     (the transposes of S and dP for KV)
//   P = exp(S - lse), dS = P o (dP - delta)
//   dQ += dS Y1                                   KV: dV += P Y2, dK += dS Y1
// and scale enters dQ and dK in fp32 at the end.
// The thread of a row of S has the row of P^T or dS that the next product takes as its TMEM
// operand, so P and dS never leave TMEM and nothing is transposed: Y1 and Y2 serve as K-major
// operands of the first products and as MN-major operands of the others. dQ and dK, dV are
// summed in two passes that each recompute S (7 products instead of 5): every sum is kept in one
// CTA's TMEM, so no fp32 gradient is accumulated in memory by atomics and results are repeatable.
// BN: streamed rows of a block; BN / 32 warpgroups share its tile, warpgroup w has columns 32 w ..
// Heads up to 64: BN 64 and two CTAs on an SM, so that one's products run while the other's warps
// wait, and one's exponentials beside the other's dS (one CTA with BN 128: 464 us for 2 x 12 heads
// of 4096 tokens, its MMA warp idle between a block's barriers). Longer heads fill TMEM: BN 128.
// TMEM: S at 0, dP at BN (P and dS over the first half of each 32 columns), accumulators behind.
constexpr int BWD_COLS = 32;
// The KV kernel's lse and delta vary along the columns of S^T, where a thread would have to fetch
// them one by one (from shared memory 1024 broadcast wavefronts a 128 x 128 tile, more than the
// products' own operands take: 303 us against 211 us without any arithmetic, 24 heads of 4096
// tokens x 64). So they enter through the products: one more step of 16 columns, in which the
// streamed side has -lse / |scale| and -delta and the kept side constants. Each value is four 16-bit
// parts of the units U = (2^15, 2^4, 2^-7, 2^-18), so nothing of fp32 is lost:
//   S^T - lse / |scale| = K Q^T + XE1 YE^T, dP^T - delta = V dO^T + XE2 YE^T,
//   YE = (parts of -lse / |scale|, parts of -delta, 0 ...), XE1 = (U, 0 ...), XE2 = (0 0 0 0, U, 0 ...).
// In fp16 the parts reach from 2^31 down to 2^-42, which covers every lse of scores that fp32 can
// tell apart (and delta alike); what lies beyond is cut to that, so that no part is ever an infinity
// or, times the other value's zeros, a NaN in every key's sums. Without swizzle, as core matrices of 8
// rows x 8 columns (128 bytes); the columns 8..15 are zeros.
// The dQ kernel leaves YE in the workspace as [batch][head][64 queries][8 rows][2 cores].
constexpr int STAT_TILE = 2048;                              // bytes of 64 queries
constexpr int XE_REGION = 128 * 16, XE_BYTES = 3 * XE_REGION;   // XE2's and XE1's first cores, zeros
__host__ __device__ constexpr int stat_tiles(int nSq) { return (nSq + 127) / 128 * 2; }
__device__ __forceinline__ uint8_t* stat_tile(const Params& p, int b, int h, int tile) {
    return p.stat + (((long long)b * p.H + h) * stat_tiles(p.Sq) + tile) * STAT_TILE;
}
// low descriptor word of an unswizzled operand; the high word: rows of cores `rows` bytes apart
__device__ __forceinline__ uint32_t desc_plain(uint32_t at, uint32_t cols) { return (at >> 4) | (cols >> 4 << 16); }
__host__ __device__ constexpr uint32_t plain_hi(uint32_t rows) { return (rows >> 4) | (1u << 14); }
// D = XE YE^T
__device__ __forceinline__ void product_plain(uint32_t leader, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .b64 a, b;\n\t.reg .pred p, q;\n\t"
        "mov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %5};\n\tsetp.ne.b32 p, 0, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(plain_hi(128)), "r"(plain_hi(256)), "r"(leader));
}
// the four parts of a value (v + more, whose sum is not rounded first) and their units: each part is
// what the ones before it left, rounded
__device__ __forceinline__ float part_unit(int i) { return i == 0 ? 0x1p15f : i == 1 ? 0x1p4f : i == 2 ? 0x1p-7f : 0x1p-18f; }
template <int DT>
__device__ __forceinline__ void four_parts(float v, float more, typename Half16<DT>::T* out) {
    using H16 = Half16<DT>;
    constexpr float MOST = 65504.f * 0x1p15f;
    if (DT == OM_DTYPE_F16 && fabsf(v) > MOST) v = copysignf(MOST, v);
    out[0] = H16::from_f((v + more) * (1.f / part_unit(0)));
    v = (v - H16::to_f(out[0]) * part_unit(0)) + more;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        out[i] = H16::from_f(v * (1.f / part_unit(i)));
        v -= H16::to_f(out[i]) * part_unit(i);
    }
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// dS is rounded to the type for its product. fp16 holds it only within 2^-14 .. 2^16 at full precision,
// and gradients come in any size, so there the kept side's row has a factor 2^a for its dS, taken back
// at the end: |dS| <= |dO_i| |V_j| + |delta_i| (Cauchy-Schwarz; P is 1 at most), and the factor brings
// the largest such bound of a row into [2^14, 2^15): no dS overflows, and those down to 2^-28 of the
// bound are normal numbers. (With the scale in dS and no factor, dO of size 1e-3 over 4096 keys left
// dQ 2 to 4 % off, and dO of size 1e-5 left nothing of it.) dQ's rows take their own |dO_i| and
// delta_i, and the largest |V_j| of the head from a launch before (vmax, per 128 keys); dK's rows take
// their own |V_j|, and from the dQ kernel the largest |dO_i| and |delta_i| of the queries that the
// CTA streams (qmax, squared and not, per 32 queries). bf16 has fp32's range and needs none of it. In
// fp16 the launch and the bounds cost 6 to 8 us of a short call: 32 x 12 heads of 197 tokens 71 -> 79 us,
// the ragged causal batch 61 -> 67, 24 heads of 4096 tokens 403 -> 413 (bf16, by the multiply that went
// and the order of the products: 403 -> 385).
struct Factor { float f, inverse; };
// P for dV is 1 at most, and in fp16 below 2^-14 no normal number (1e-7 came out up to 30 % off, and
// with it the dV of a key that every query gives so little): there the dK/dV kernel works with 2^14 P,
// by 14 more in the exponent that its parts of -lse give (by a sum per score: 24 heads of 4096 tokens
// 417 -> 423 us).
template <int DT> constexpr int P_SHIFT = DT == OM_DTYPE_F16 ? 14 : 0;
__device__ __forceinline__ Factor range_factor(float bound) {
    if (!(bound >= 0x1p-100f && bound <= 0x1p100f)) return {1.f, 1.f};   // no gradient, or not finite
    const int e = __float_as_int(bound) >> 23;
    return {__int_as_float((2 * 127 + 14 - e) << 23), __int_as_float((e - 14) << 23)};
}
// the largest of the lanes' values, none of which is negative
__device__ __forceinline__ float warp_max(float v) { return __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(v))); }
__device__ __forceinline__ float if_finite(float v) { return v < INFINITY ? v : 0.f; }
template <int DT>
__device__ __forceinline__ float squares(const uint4& u) {
    const auto* v = reinterpret_cast<const typename Half16<DT>::T2*>(&u);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = Half16<DT>::unpack(v[i]);
        s += f.x * f.x + f.y * f.y;
    }
    return s;
}
// vmax: the largest sum of squares of a value row of 128 keys, rows that are not finite left out. 8 or
// 16 lanes a row, one 16-byte load each, 32 rows at a time; all of a thread's loads go out before anything waits (one after
// another, behind the length, they took 8 us of an idle GPU's time instead of 5)
template <int DT>
__global__ void __launch_bounds__(512) value_norms_kernel(const Params p) {
    __shared__ float sh[16];
    pdl_launch_dependents();
    const int tiles = (p.Sk + 127) / 128, t0 = blockIdx.x % tiles * 128, bh = blockIdx.x / tiles;
    const int b = bh / p.Hkv, h = bh - b * p.Hkv, end = len_of(p.kvlens, b, p.Sk);
    const int wide = blockDim.x / 32, col = threadIdx.x % wide * 8, r = threadIdx.x / wide;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = r + i * 32;
        v[i] = make_uint4(0, 0, 0, 0);
        if (t0 + t < p.Sk && col < p.D)
            v[i] = __ldg(reinterpret_cast<const uint4*>(row<DT>(p.v, b, t0 + t, h) + col));
    }
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float s = squares<DT>(v[i]);
        for (int o = wide / 2; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        if (t0 + r + i * 32 < end) most = fmaxf(most, if_finite(s));
    }
    most = warp_max(most);
    if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = most;
    __syncthreads();
    if (threadIdx.x < 32) {
        most = warp_max(threadIdx.x < wide ? sh[threadIdx.x] : 0.f);
        if (threadIdx.x == 0) p.vmax[blockIdx.x] = most;
    }
}
constexpr int max_of(int a, int b) { return a > b ? a : b; }
template <int DP>
struct BwdCfg {
    static constexpr int BN = DP == 64 ? 64 : 128, OCC = DP == 64 ? 2 : 1;
    static constexpr int WG = BN / BWD_COLS, THREADS = WG * 128 + 64;
    static constexpr int TILE = DP / 64 * PANEL, Y_TILE = DP / 64 * BN * 128;
    static constexpr int SLOTS = DP == 64 ? 8 : 4;
    static constexpr int Y_OFF = 2 * TILE;
    static constexpr int STAT = BN / 64 * STAT_TILE;         // YE of a block, per pair of slots
    static constexpr int STAT_OFF = Y_OFF + SLOTS * Y_TILE;
    static constexpr int XE_OFF = STAT_OFF + max_of(SLOTS / 2 * STAT, WG * 128 * 8);
    static constexpr int BAR_OFF = XE_OFF + XE_BYTES;
    static constexpr int SMEM = BAR_OFF + 512;
    static constexpr int DP_COL = BN, ACC = 2 * BN, TMEM_COLS = 2 * BN + 2 * DP;
    static_assert(TMEM_COLS * OCC <= 512 && (SMEM + 1024) * OCC <= 228 * 1024, "on-chip memory");
};

template <int DP, bool KV, int DT>
__global__ void __launch_bounds__(BwdCfg<DP>::THREADS, BwdCfg<DP>::OCC)
attn_bwd_kernel(const __grid_constant__ CUtensorMap mx1, const __grid_constant__ CUtensorMap mx2,
                const __grid_constant__ CUtensorMap my1, const __grid_constant__ CUtensorMap my2,
                const __grid_constant__ CUtensorMap mo1, const __grid_constant__ CUtensorMap mo2, const Params p) {
    using Cf = BwdCfg<DP>;
    // aligned by its declaration, so that every address below is a constant (rounded up at run time,
    // the barriers' pointers took the registers that the scores need)
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) % 1024) {
        if (threadIdx.x == 0) atomicOr(p.err, ERR_LOAD);
        return;
    }
    float* stat = reinterpret_cast<float*>(smem + Cf::STAT_OFF);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cf::BAR_OFF);
    uint64_t *x_full = bars, *s_full = bars + 1, *dp_full = bars + 2, *acc_full = bars + 3, *drain = bars + 4,
             *p_ready = bars + 5, *ds_ready = bars + 6, *out_ready = bars + 7;
    uint64_t* full = bars + 8;
    uint64_t* empty = full + Cf::SLOTS;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(empty + Cf::SLOTS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

    const int warp = uniform(threadIdx.x / 32), lane = threadIdx.x % 32;
    constexpr int W_LOAD = Cf::WG * 4, W_MMA = W_LOAD + 1, CW = BWD_COLS, BN = Cf::BN;
    const int rep = p.H / p.Hkv, heads = KV ? p.Hkv : p.H;
    // causal: heads fastest and the tiles with the longest rows (first columns) first
    const int tiles = ((KV ? p.Sk : p.Sq) + 127) / 128, bhs = p.B * heads;
    const int split = blockIdx.x % p.splits, cta = blockIdx.x / p.splits;
    const int bh = p.causal ? cta % bhs : cta / tiles;
    const int tile_x = p.causal ? cta / bhs : cta % tiles;
    const int hx = bh % heads, b = bh / heads;                   // head of the kept tiles
    const int hy0 = KV ? hx * rep : hx / rep;                    // first head of the streamed ones
    const int r0 = (p.causal && !KV ? tiles - 1 - tile_x : tile_x) * 128;
    const int ql = len_of(p.qlens, b, p.Sq), kl = len_of(p.kvlens, b, p.Sk);
    // streamed blocks: first .. first + per of each streamed head
    int first = 0, per = 0;
    if (KV) {
        if (r0 < kl) {
            first = p.causal ? max(0, r0 - (kl - ql)) / BN : 0;
            per = max(0, (ql + BN - 1) / BN - first);
        }
    } else {
        int end = r0 < ql ? kl : 0;
        if (p.causal) end = min(end, min(r0 + 128, ql) + kl - ql);
        per = end > 0 ? (end + BN - 1) / BN : 0;
    }
    // this part's share of them, from the it0-th on (KV: head by head)
    const int all = KV ? per * rep : per, share = (all + p.splits - 1) / p.splits, it0 = split * share;
    const int nblk = uniform(max(0, min(all - it0, share)));
    const int y_start = per > 0 ? first + it0 % per : 0, hy_start = hy0 + (per > 0 ? it0 / per : 0);

    if (threadIdx.x == 0) {
        for (int i = 0; i < 8; ++i) mbar_init(bars + i, i < 5 ? 1 : Cf::WG * 4);
        for (int i = 0; i < Cf::SLOTS; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_holder)), "r"(Cf::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // dQ: a thread's part of its row's delta, 8 elements of dO . O at a time, and the row's lse,
    // fetched while the barriers and TMEM are set up
    constexpr bool F16 = DT == OM_DTYPE_F16;
    float delta_part = 0.f, grad_part = 0.f, lse_in = 0.f;
    if (!KV && warp < W_LOAD) {
        const int w = warp / 4, r = r0 + (warp % 4) * 32 + lane;
        if (r < ql) {
            const auto* go = attn::row<DT>(p.dout, b, r, hx);
            const auto* o = attn::row<DT>(p.o, b, r, hx);
            constexpr int N = DP / 8 / Cf::WG;
            uint4 u[N], v[N];
#pragma unroll
            for (int x = 0; x < N; ++x)
                if ((w + x * Cf::WG) * 8 < p.D) {
                    u[x] = __ldg(reinterpret_cast<const uint4*>(go) + w + x * Cf::WG);
                    v[x] = __ldg(reinterpret_cast<const uint4*>(o) + w + x * Cf::WG);
                }
            lse_in = __ldg(p.lse + ((long long)b * p.H + hx) * p.Sq + r);
#pragma unroll
            for (int x = 0; x < N; ++x)
                if ((w + x * Cf::WG) * 8 < p.D) {
                    const auto* a2 = reinterpret_cast<const typename Half16<DT>::T2*>(&u[x]);
                    const auto* b2 = reinterpret_cast<const typename Half16<DT>::T2*>(&v[x]);
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const float2 f = Half16<DT>::unpack(a2[y]), g = Half16<DT>::unpack(b2[y]);
                        delta_part += f.x * g.x + f.y * g.y;
                    }
                    if (F16) grad_part += squares<DT>(u[x]);
                }
        }
    }
    if (KV) {                             // the constant operands, 8 columns of a row at a time
        for (int i = threadIdx.x; i < XE_BYTES / 16; i += Cf::THREADS) {
            alignas(16) typename Half16<DT>::T v[8];
            const int region = i / 128;   // 0: XE2, 1: XE1, 2: zeros
            for (int c = 0; c < 8; ++c) v[c] = Half16<DT>::from_f(region + c / 4 == 1 ? part_unit(c % 4) : 0.f);
            reinterpret_cast<uint4*>(smem + Cf::XE_OFF)[i] = *reinterpret_cast<const uint4*>(v);
        }
        fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(*tmem_holder);
    if (!KV) pdl_launch_dependents();     // the KV kernel may set up where this one's CTAs have left
    unsigned int err = 0;

    if (warp == W_LOAD) {
        if (lane == 0 && nblk > 0) {
            mbar_expect_tx(x_full, 2 * Cf::TILE);
            load_tile<DP>(0, smem, &mx1, x_full, r0, hx, b);
            load_tile<DP>(Cf::TILE, smem, &mx2, x_full, r0, hx, b);
            int i = 0, y = y_start, hy = hy_start;
            for (; i < 2 * nblk; ++i) {   // Y1 (KV: and its queries' statistics), Y2 of each block in turn
                const int slot = i % Cf::SLOTS;
                if (!mbar_wait(empty + slot, ((i / Cf::SLOTS) & 1) ^ 1, abort_flag)) { err = ERR_LOAD; break; }
                mbar_expect_tx(full + slot, Cf::Y_TILE + (KV && !(i & 1) ? Cf::STAT : 0));
                if (KV && i == 0) pdl_wait();     // the dQ kernel's statistics
                if (KV && !(i & 1))
                    bulk_load(smem + Cf::STAT_OFF + slot / 2 * Cf::STAT, stat_tile(p, b, hy, y * (BN / 64)), Cf::STAT,
                              full + slot);
                load_tile<DP, BN>(Cf::Y_OFF + slot * Cf::Y_TILE, smem, i & 1 ? &my2 : &my1, full + slot, y * BN, hy, b);
                if (i & 1 && ++y == first + per) { y = first; ++hy; }
            }
            if (err || *abort_flag) {     // every load issued has to land before the CTA ends
                *abort_flag = 1;
                if (!mbar_wait_drain(x_full, 0)) err |= ERR_DRAIN;
                for (int j = max(0, i - Cf::SLOTS); j < i; ++j)
                    if (!mbar_wait_drain(full + j % Cf::SLOTS, (j / Cf::SLOTS) & 1)) err |= ERR_DRAIN;
            }
        }
    } else if (warp == W_MMA) {
        if (nblk > 0) {
            const uint32_t leader = elect();
            const int ks = (p.D + 15) / 16;
            const bool f16 = DT == OM_DTYPE_F16;
            const uint32_t id_s = idesc_f16(f16, BN, false, p.neg), id_dp = idesc_f16(f16, BN, false, false);
            const uint32_t id_acc = idesc_f16(f16, ks * 16, true, false);
            const uint32_t x1 = smem_u32(smem), x2 = x1 + Cf::TILE, y = x1 + Cf::Y_OFF;
            const uint32_t xe = x1 + Cf::XE_OFF, ye = x1 + Cf::STAT_OFF;
            auto tile = [&](int i) { return y + (i % Cf::SLOTS) * Cf::Y_TILE; };
            auto wait_y = [&](int i) { return warp_wait(full + i % Cf::SLOTS, (i / Cf::SLOTS) & 1, abort_flag); };
            auto score = [&](uint32_t d, uint32_t x, int i, uint32_t id, uint64_t* bar) {
                tc_fence_after();
                // first the statistics, so that the sum over the head dimension runs towards the small
                // difference and not the other way (the sums drop bits below their largest term's)
                if (KV)                   // d == 0: XE1, else XE2
                    product_plain(leader, tmem + d, desc_plain(xe + (d ? 0 : XE_REGION), d ? 2 * XE_REGION : XE_REGION),
                                  desc_plain(ye + i / 2 % (Cf::SLOTS / 2) * Cf::STAT, 128), id_dp);
                product_k<DP, BN, KV>(leader, tmem + d, x, tile(i), id, ks);
                commit(leader, bar);
            };
            bool ok = warp_wait(x_full, 0, abort_flag) && wait_y(0);
            if (ok) {
                score(0, x1, 0, id_s, s_full);
                ok = wait_y(1);
            }
            if (ok) score(Cf::DP_COL, x2, 1, id_dp, dp_full);
            for (int i = 0; ok && i < nblk; ++i) {
                // products run in the order of their issue: S of the next block may overwrite P
                // right behind the product that reads it, and dP its dS
                const bool more = i + 1 < nblk;
                ok = (!more || wait_y(2 * i + 2)) && warp_wait(p_ready, i & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                if (KV) product_mn<CW, BN>(leader, tmem + Cf::ACC + DP, tmem, tile(2 * i + 1), id_acc, i > 0);
                if (more) score(0, x1, 2 * i + 2, id_s, s_full);
                ok = (!more || wait_y(2 * i + 3)) && warp_wait(ds_ready, i & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                product_mn<CW, BN>(leader, tmem + Cf::ACC, tmem + Cf::DP_COL, tile(2 * i), id_acc, i > 0);
                commit(leader, empty + (2 * i) % Cf::SLOTS);
                commit(leader, empty + (2 * i + 1) % Cf::SLOTS);
                if (more)
                    score(Cf::DP_COL, x2, 2 * i + 3, id_dp, dp_full);
                else
                    commit(leader, acc_full);
            }
            if (!ok) {                    // no MMA may run on when the CTA ends
                *abort_flag = 1;
                err = ERR_MMA;
                commit(leader, drain);
                if (!mbar_wait_drain(drain, 0)) err |= ERR_DRAIN;
            }
        }
    } else {
        const int w = warp / 4, row = (warp % 4) * 32 + lane, tid = threadIdx.x;
        const int r = r0 + row;
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;
        const uint32_t s_addr = tmem + lanes + w * CW, dp_addr = s_addr + Cf::DP_COL;
        constexpr float LOG2E = 1.4426950408889634f;
        bool ok = true;
        float lse2 = 0.f, ds0 = 0.f;          // dQ: the row's -lse * log2(e) and -delta (times its factor)
        Factor range = {1.f, 1.f};
        int row_lo = 0, row_hi = 0;           // the streamed rows that this row meets
        if (KV) {
            if (r < kl) {
                row_lo = p.causal ? max(0, r - (kl - ql)) : 0;
                row_hi = ql;
            }
        } else {
            row_hi = r < ql ? kl : 0;
            if (p.causal) row_hi = min(row_hi, r + kl - ql + 1);
            if (row_hi > 0) lse2 = -lse_in * LOG2E;
            stat[tid] = row_hi > 0 ? delta_part : 0.f;
            if (F16) stat[Cf::WG * 128 + tid] = row_hi > 0 ? grad_part : 0.f;
            warp_arrive(out_ready);               // its first phase: the parts of delta
            ok = warp_wait(out_ready, 0, abort_flag);
            float delta = 0.f, grad = 0.f;
            for (int x = 0; x < Cf::WG; ++x) {
                delta += stat[row + x * 128];
                if (F16) grad += stat[(Cf::WG + x) * 128 + row];
            }
            if (F16) {
                pdl_wait();                       // vmax
                const int tiles = (p.Sk + 127) / 128;
                const float* v = p.vmax + ((long long)b * p.Hkv + hy0) * tiles;
                float most = 0.f;
                for (int x = lane; x < tiles; x += 32) most = fmaxf(most, __ldcg(v + x));
                range = range_factor(sqrtf(grad) * sqrtf(warp_max(most)) + fabsf(delta));
            }
            ds0 = -delta * range.f;
            if (ok && w == 0 && split == 0) {   // for the KV kernel
                alignas(16) typename Half16<DT>::T v[8];
                four_parts<DT>(row_hi > 0 ? -lse_in * p.inv_scale : 0.f, P_SHIFT<DT> / p.scale2, v);
                four_parts<DT>(-delta, 0.f, v + 4);
                uint4* out = reinterpret_cast<uint4*>(stat_tile(p, b, hx, (r0 + row) / 64) + row % 64 / 8 * 256 + row % 8 * 16);
                out[0] = *reinterpret_cast<const uint4*>(v);
                out[8] = make_uint4(0, 0, 0, 0);
                if (F16) {
                    const float2 most = {warp_max(if_finite(grad)), warp_max(if_finite(fabsf(delta)))};
                    if (lane == 0) p.qmax[((long long)b * p.H + hx) * stat_tiles(p.Sq) * 2 + (r0 + row) / 32] = most;
                }
            }
        }
        if (KV && F16 && nblk > 0) {
            pdl_wait();                           // qmax
            float2 most = {0.f, 0.f};
            for (int h = 0; h < rep; ++h) {
                const float2* q = p.qmax + ((long long)b * p.H + hy0 + h) * stat_tiles(p.Sq) * 2;
                for (int x = first * BN / 32 + lane; x < (first + per) * BN / 32; x += 32) {
                    const float2 v = __ldcg(q + x);
                    most = {fmaxf(most.x, v.x), fmaxf(most.y, v.y)};
                }
            }
            most = {warp_max(most.x), warp_max(most.y)};
            ok = warp_wait(x_full, 0, abort_flag);
            float v2 = 0.f;                       // |V_j|^2 from the kept tile, its columns in any order
#pragma unroll
            for (int x = 0; x < DP / 8; ++x)
                v2 += squares<DT>(*reinterpret_cast<const uint4*>(smem + Cf::TILE + x / 8 * PANEL + row * 128 + ((x ^ row) % 8 << 4)));
            range = range_factor(sqrtf(most.x) * sqrtf(v2) + most.y);
            range.f *= 1.f / (1 << P_SHIFT<DT>);
        }
        int y0 = y_start * BN;
        for (int i = 0; ok && i < nblk; ++i) {
            ok = warp_wait(s_full, i & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            uint32_t pv[CW];
            tmem_ld32_issue(s_addr, pv);
            tmem_ld_wait<CW>(pv);
            float* pr = reinterpret_cast<float*>(pv);
            if (!KV) {                        // S may be overwritten: P stays in registers
                tc_fence_before();
                warp_arrive(p_ready);
            }
            const int lo = row_lo - y0 - w * CW, hi = row_hi - y0 - w * CW;
            const bool mask = __any_sync(~0u, lo > 0 || hi < CW);
            const bool some = __any_sync(~0u, max(lo, 0) < min(hi, CW));
            if (some) {
#pragma unroll
                for (int c = 0; c < CW; c += 2) {
                    const F2 v = {pr[c], pr[c + 1]}, k = {p.scale2, p.scale2};
                    const F2 e = KV ? mul2(v, k) : fma2(v, k, {lse2, lse2});
                    pr[c] = ex2(e.x);
                    pr[c + 1] = ex2(e.y);
                }
            }
            if (mask) {
#pragma unroll
                for (int c = 0; c < CW; ++c) pr[c] = c >= lo && c < hi ? pr[c] : 0.f;
            }
            // streamed rows past the sequence's length may hold anything
            const int y_end = KV ? ql : kl;
            if (w < 2 && y_end - y0 < BN) {
                const int iy = 2 * i + w;
                ok = warp_wait(full + iy % Cf::SLOTS, (iy / Cf::SLOTS) & 1, abort_flag);
                if (!ok) break;
                zero_tail<DP, BN>(smem + Cf::Y_OFF + iy % Cf::SLOTS * Cf::Y_TILE, y_end - y0, row);
            }
            if (KV) {
                uint32_t pk[CW / 2];
#pragma unroll
                for (int c = 0; c < CW / 2; ++c) pk[c] = pack16<DT>(pr[2 * c], pr[2 * c + 1]);
                tmem_st16(s_addr, pk);
                tmem_st_wait();
                tc_fence_before();
                warp_arrive(p_ready);
            }
            ok = warp_wait(dp_full, i & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            uint32_t dv[CW], dk[CW / 2];
            tmem_ld32_issue(dp_addr, dv);
            tmem_ld_wait<CW>(dv);
            float* dp = reinterpret_cast<float*>(dv);
#pragma unroll
            for (int c = 0; c < CW; c += 2) {
                const F2 v = {dp[c], dp[c + 1]}, k = {range.f, range.f};
                const F2 e = mul2({pr[c], pr[c + 1]}, KV ? (F16 ? mul2(v, k) : v) : F16 ? fma2(v, k, {ds0, ds0}) : add2(v, {ds0, ds0}));
                dp[c] = e.x;
                dp[c + 1] = e.y;
            }
            if (mask) {                       // 0 * what a masked place holds
#pragma unroll
                for (int c = 0; c < CW; ++c) dp[c] = c >= lo && c < hi ? dp[c] : 0.f;
            }
#pragma unroll
            for (int c = 0; c < CW / 2; ++c) dk[c] = pack16<DT>(dp[2 * c], dp[2 * c + 1]);
            tmem_st16(dp_addr, dk);
            tmem_st_wait();
            tc_fence_before();
            warp_arrive(ds_ready);
            y0 += BN;
            if (KV && y0 == (first + per) * BN) y0 = first * BN;
        }
        if (ok && nblk > 0) ok = warp_wait(acc_full, 0, abort_flag);
        if (!ok) {
            *abort_flag = 1;
            err = ERR_MATH;
        } else {
            tc_fence_after();
            // the warpgroups take alternate 32 columns; KV: the first half of them dK, the others dV
            constexpr int HALF = Cf::WG / 2;
            const int rows = KV ? p.Sk : p.Sq;
            uint8_t* tile = smem + (KV && w >= HALF ? Cf::TILE : 0);   // X's, which every product has read
            // partial dV behind all of dK's
            float* part = r < rows && p.splits > 1
                              ? p.part + ((((KV && w >= HALF ? p.splits : 0) + (long long)split) * bhs + bh) * rows + r) * p.D
                              : nullptr;
            const uint32_t acc = tmem + lanes + Cf::ACC + (KV ? w / HALF * DP : 0);
            const float f = KV && w >= HALF ? 1.f / (1 << P_SHIFT<DT>) : p.scale * range.inverse;
            for (int c = (KV ? w % HALF : w) * 32; c < p.D; c += (KV ? HALF : Cf::WG) * 32) {
                uint32_t o[32];
                if (nblk > 0) {
                    tmem_ld32_issue(acc + c, o);
                    tmem_ld_wait<32>(o);
                }
                store_chunk<DT>(o, nblk > 0, f, p.splits > 1, tile, row, part, c, p.D);
            }
            if (p.splits == 1) {
                fence_async_smem();
                warp_arrive(out_ready);
                if (warp == 0) {
                    if (!warp_wait(out_ready, KV ? 0 : 1, abort_flag)) {
                        err = ERR_MATH;
                    } else if (lane == 0) {
                        store_tile(&mo1, smem, p.D, r0, hx, b);
                        if (KV) store_tile(&mo2, smem + Cf::TILE, p.D, r0, hx, b);
                        bulk_commit();
                        bulk_wait_read<0>();
                    }
                }
            }
        }
    }
    if (err) atomicOr(p.err, err);
    if (KV && nblk == 0) pdl_wait();      // so that this kernel's end means the dQ kernel's end too
    tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cf::TMEM_COLS));
    }
}

// ---------------------------------------------------------------- joining parts
// One warp per row of [batch][head][token]: the parts in a fixed order. LSE: each weighted by 2^(its
// log2 sum - the largest), their sum of weights into lse; else their sum.
template <int DT, bool LSE>
__global__ void __launch_bounds__(128) join_kernel(const Params p, const View out0, const View out1, int T, int H) {
    const int lane = threadIdx.x % 32;
    const long long row = blockIdx.x * 4LL + threadIdx.x / 32, rows = (long long)p.B * H * T;
    if (row >= rows) return;
    const View& out = blockIdx.y ? out1 : out0;
    const float* part = p.part + (blockIdx.y ? p.splits * rows * p.D : 0);
    const int t = (int)(row % T), h = (int)(row / T % H), b = (int)(row / T / H);
    // lanes: `wide` float4 columns x 32 / wide parts at a time
    const int cols = p.D / 4, wide = cols <= 2 ? 2 : cols <= 4 ? 4 : cols <= 8 ? 8 : cols <= 16 ? 16 : 32;
    const int col = lane % wide, first = lane / wide, step = 32 / wide;
    float top = -INFINITY, total = 0.f;
    if (LSE) {
        for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, p.part_lse[s * rows + row]);
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = first; s < p.splits; s += step) {
        float w = 1.f;
        if (LSE) {                                // 0 where the part saw no key; its row is zeros
            const float l = p.part_lse[s * rows + row];
            w = l == -INFINITY ? 0.f : exp2f(l - top);
            total += w;
        }
        const float4 v = col < cols ? *reinterpret_cast<const float4*>(part + (s * rows + row) * p.D + col * 4)
                                    : make_float4(0.f, 0.f, 0.f, 0.f);
        acc = make_float4(fmaf(w, v.x, acc.x), fmaf(w, v.y, acc.y), fmaf(w, v.z, acc.z), fmaf(w, v.w, acc.w));
    }
    for (int o = 16; o >= wide; o >>= 1) {
        acc.x += __shfl_xor_sync(~0u, acc.x, o);
        acc.y += __shfl_xor_sync(~0u, acc.y, o);
        acc.z += __shfl_xor_sync(~0u, acc.z, o);
        acc.w += __shfl_xor_sync(~0u, acc.w, o);
        if (LSE) total += __shfl_xor_sync(~0u, total, o);
    }
    const float f = !LSE ? 1.f : total == 0.f ? 0.f : 1.f / total;
    if (lane < cols)
        *reinterpret_cast<uint2*>(row_out<DT>(out, b, t, h) + lane * 4) =
            make_uint2(pack16<DT>(acc.x * f, acc.y * f), pack16<DT>(acc.z * f, acc.w * f));
    if (LSE && lane == 0 && p.lse) p.lse[row] = total == 0.f ? -INFINITY : (top + log2f(total)) * LN2;
}
template <int DT, bool LSE>
static int join(DeviceCtx* c, const Params& p, const View& out, int T, int H, const View* second = nullptr) {
    const long long blocks = ((long long)p.B * H * T + 3) / 4;
    if (blocks > 0x7FFFFFFF) return OM_ERR_UNSUPPORTED;
    join_kernel<DT, LSE><<<dim3((unsigned)blocks, second ? 2 : 1), 128, 0, c->compute>>>(p, out, second ? *second : out, T, H);
    return after_launch(c);
}

// Parts of the streamed axis for `ctas` tiles of `blocks` blocks each (causal: half of that on the
// average), on `places` of CTAs, 148 SMs times the CTAs that an SM holds: the count with the least
// estimated time, in blocks: the longest part or the even share of all of them, each part with about
// 4 blocks' time for its start and end; joining costs about 3 (another launch) and grows with the
// parts. Parts of two blocks at least. (84 tiles of 28 causal blocks: 3 parts, 62 -> 32 us; 16 tiles
// of 32 blocks: 16 parts, 55 -> 18 us: the constants come from these two.) The forward's blocks count
// as 128 keys, also where it takes two of 64; lengths are on the device and count as full. The number
// of SMs is a constant, as the workspace's size has to be the same without a device to ask.
static int parts(long long ctas, int blocks, int places, bool causal) {
    int best = 1;
    float least = INFINITY;
    for (int n = 1; n <= 64 && (n == 1 || n * 2 <= blocks); ++n) {
        const float mean = (causal ? 0.5f : 1.f) * blocks / n + 4.f, rounds = (float)(ctas * n) / places;
        const float t = fmaxf((float)blocks / n + 4.f, (causal ? rounds : ceilf(rounds)) * mean) + (n > 1 ? 3.f + 0.1f * n : 0.f);
        if (t < least) { least = t; best = n; }
    }
    return best;
}
// The split of each kernel of a problem and the workspace it takes.
struct Plan {
    int nt, fwd, dq, dkv;                 // query tiles of a forward CTA; parts
    long long fwd_bytes, bwd_bytes, qmax_at, vmax_at, dq_at, dkv_at;
};
static Plan plan(int B, int H, int Hkv, int Sq, int Sk, int D, bool causal) {
    Plan n;
    const long long qt = (Sq + 127) / 128, kt = (Sk + 127) / 128, bh = (long long)B * H, bhk = (long long)B * Hkv;
    n.nt = Sq <= 128 ? 1 : 2;
    n.fwd = parts((qt + n.nt - 1) / n.nt * bh, (int)kt, n.nt == 1 ? 296 : 148, causal);
    n.fwd_bytes = n.fwd > 1 ? n.fwd * bh * Sq * (D + 1) * 4 : 0;
    const int places = D <= 64 ? 296 : 148, bn = D <= 64 ? 64 : 128;
    n.dq = parts(qt * bh, (Sk + bn - 1) / bn, places, causal);
    n.dkv = parts(kt * bhk, (Sq + bn - 1) / bn * (H / Hkv), places, causal);
    n.qmax_at = bh * stat_tiles(Sq) * STAT_TILE;
    n.vmax_at = n.qmax_at + bh * stat_tiles(Sq) * 2 * (long long)sizeof(float2);
    n.dq_at = n.vmax_at + (bhk * kt * 4 + 15) / 16 * 16;
    n.dkv_at = n.dq_at + (n.dq > 1 ? n.dq * bh * Sq * D * 4 : 0);
    n.bwd_bytes = n.dkv_at + (n.dkv > 1 ? 2 * n.dkv * bhk * Sk * D * 4 : 0);
    return n;
}

static int check_sizes(int nBatch, int nHeads, int nKvHeads, int nSq, int nSk, int nHeadDim) {
    if (nBatch < 0 || nHeads <= 0 || nKvHeads <= 0 || nHeads % nKvHeads || nSq < 0 || nSk < 0 ||
        nHeadDim <= 0)
        return OM_ERR_INVALID;
    if (nHeadDim % 8 || nHeadDim > 128)
        return OM_ERR_UNSUPPORTED;
    return OM_OK;
}

// The view of one tensor; false for a null or misaligned pointer or a stride the kernels do not
// take. Dimensions of length 1 may have any stride; a tensor without elements may be null.
static bool view(View* v, const void* p, const long long* s, int nB, int nT, int nH) {
    v->p = const_cast<void*>(p);
    v->sb = s[0]; v->st = s[1]; v->sh = s[2];
    if (nB == 0 || nT == 0) return true;
    if (!p || reinterpret_cast<uintptr_t>(p) % 16) return false;
    const int len[3] = {nB, nT, nH};
    for (int i = 0; i < 3; ++i)
        if (len[i] > 1 && (s[i] <= 0 || s[i] % 8)) return false;
    return true;
}

static void set_scale(Params* p, float scale) {
    p->scale = scale;
    p->neg = scale < 0.f;
    p->scale2 = fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f);
    p->inv_scale = 1.f / fabsf(scale);
}

// A tensor map over a [batch, token, head, D] view with boxes of 64 columns x `rows` tokens.
// Strides of dimensions of length 1 are replaced by one that the map takes.
static int encode(CUtensorMap* map, const View& v, int nB, int nT, int nH, int D, int dt, int rows = 128) {
    PFN_cuTensorMapEncodeTiled_v12000 fn = tc::encode_tiled_fn();
    if (!fn) return OM_ERR_DRIVER;
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)nT, (cuuint64_t)nH, (cuuint64_t)nB};
    cuuint64_t strides[3] = {nT > 1 ? (cuuint64_t)v.st * 2 : 256, nH > 1 ? (cuuint64_t)v.sh * 2 : 256,
                             nB > 1 ? (cuuint64_t)v.sb * 2 : 256};
    cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, dt == OM_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                          4, v.p, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? OM_OK : OM_ERR_INVALID;
}

template <int DP, int NT, int DT>
static int launch_fwd(DeviceCtx* c, const Params& p) {
    using Cf = FwdCfg<DP, NT>;
    auto kern = attn_fwd_kernel<DP, NT, DT>;
    static bool attr_set[64] = {false};
    if (!attr_set[c->device]) {
        cudaFuncAttributes fa;
        OMB_CHECK(cudaFuncGetAttributes(&fa, kern));
        if (fa.numRegs < Cf::LAUNCH_REGS) return OM_ERR_UNSUPPORTED;   // built with other limits
        OMB_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cf::SMEM));
        attr_set[c->device] = true;
    }
    CUtensorMap mq = {}, mk = {}, mv = {}, mo = {};
    int st = encode(&mq, p.q, p.B, p.Sq, p.H, p.D, DT);
    if (st == OM_OK && p.Sk > 0) st = encode(&mk, p.k, p.B, p.Sk, p.Hkv, p.D, DT, Cf::KB);
    if (st == OM_OK && p.Sk > 0) st = encode(&mv, p.v, p.B, p.Sk, p.Hkv, p.D, DT, Cf::KB);
    if (st == OM_OK && p.splits == 1) st = encode(&mo, p.o, p.B, p.Sq, p.H, p.D, DT);
    if (st != OM_OK) return st;
    const long long items = (long long)((p.Sq + NT * 128 - 1) / (NT * 128)) * p.B * p.H * p.splits;
    if (items > 0x7FFF0000) return OM_ERR_UNSUPPORTED;
    const int tiles = (p.Sq + NT * 128 - 1) / (NT * 128);
    Params q = p;
    q.items = (int)items;
    q.by_splits = div_by(p.splits);
    q.by_fast = div_by(p.causal ? p.B * p.H : tiles);
    q.by_heads = div_by(p.H);
    const int places = c->num_sms * Cf::OCC, grid = q.items < places ? q.items : places;
    kern<<<grid, Cf::THREADS, Cf::SMEM, c->compute>>>(mq, mk, mv, mo, q);
    return after_launch(c);
}
template <int DT>
static int forward(DeviceCtx* c, Params p, void* workspace) {
    const Plan n = plan(p.B, p.H, p.Hkv, p.Sq, p.Sk, p.D, p.causal);
    p.splits = n.fwd;
    p.part = static_cast<float*>(workspace);
    p.part_lse = p.part + (long long)n.fwd * p.B * p.H * p.Sq * p.D;
    if (n.fwd > 1 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16)) return OM_ERR_INVALID;
    int st;
    if (p.D <= 64)
        st = n.nt == 1 ? launch_fwd<64, 1, DT>(c, p) : launch_fwd<64, 2, DT>(c, p);
    else
        st = n.nt == 1 ? launch_fwd<128, 1, DT>(c, p) : launch_fwd<128, 2, DT>(c, p);
    return st == OM_OK && n.fwd > 1 ? join<DT, true>(c, p, p.o, p.Sq, p.H) : st;
}

// x1, x2: maps of the kept tiles (128 rows), y1, y2: of the streamed ones (BN rows)
template <int DP, bool KV, int DT>
static int launch_bwd(DeviceCtx* c, const CUtensorMap& x1, const CUtensorMap& x2, const CUtensorMap& y1,
                      const CUtensorMap& y2, const Params& p, bool overlap) {
    using Cf = BwdCfg<DP>;
    CUtensorMap o1 = {}, o2 = {};         // dQ, or dK and dV
    if (p.splits == 1) {
        const int T = KV ? p.Sk : p.Sq, H = KV ? p.Hkv : p.H;
        int st = encode(&o1, KV ? p.dk : p.dq, p.B, T, H, p.D, DT);
        if (st == OM_OK && KV) st = encode(&o2, p.dv, p.B, T, H, p.D, DT);
        if (st != OM_OK) return st;
    }
    auto kern = attn_bwd_kernel<DP, KV, DT>;
    static bool attr_set[64] = {false};
    if (!attr_set[c->device]) {
        OMB_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cf::SMEM));
        attr_set[c->device] = true;
    }
    const long long n = (long long)(((KV ? p.Sk : p.Sq) + 127) / 128) * p.B * (KV ? p.Hkv : p.H) * p.splits;
    if (n > 0x7FFFFFFF) return OM_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n);
    cfg.blockDim = dim3(Cf::THREADS);
    cfg.dynamicSmemBytes = Cf::SMEM;
    cfg.stream = c->compute;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = overlap ? 1 : 0;           // it may set up while the launch before it ends
    OMB_CHECK(cudaLaunchKernelEx(&cfg, kern, x1, x2, y1, y2, o1, o2, p));
    return after_launch(c);
}
template <int DP, int DT>
static int backward(DeviceCtx* c, Params p) {
    constexpr int BN = BwdCfg<DP>::BN;
    CUtensorMap m[2][4] = {};             // Q, K, V, dO; boxes of 128 and of BN rows
    const View* view[4] = {&p.q, &p.k, &p.v, &p.dout};
    for (int i = 0; i < 4; ++i) {
        const bool kv = i == 1 || i == 2;
        if ((kv ? p.Sk : p.Sq) == 0) continue;
        for (int r = 0; r < 2; ++r) {
            const int st = encode(&m[r][i], *view[i], p.B, kv ? p.Sk : p.Sq, kv ? p.Hkv : p.H, p.D, DT, r ? BN : 128);
            if (st != OM_OK) return st;
        }
    }
    const Plan n = plan(p.B, p.H, p.Hkv, p.Sq, p.Sk, p.D, p.causal);
    int st = OM_OK;
    const bool norms = DT == OM_DTYPE_F16 && p.Sq > 0 && p.Sk > 0;
    p.qmax = reinterpret_cast<float2*>(p.stat + n.qmax_at);
    p.vmax = reinterpret_cast<float*>(p.stat + n.vmax_at);
    if (norms) {
        const long long blocks = (long long)p.B * p.Hkv * ((p.Sk + 127) / 128);
        if (blocks > 0x7FFFFFFF) return OM_ERR_UNSUPPORTED;
        value_norms_kernel<DT><<<(unsigned)blocks, p.D <= 64 ? 256 : 512, 0, c->compute>>>(p);
        st = after_launch(c);
        if (st != OM_OK) return st;
    }
    if (p.Sq > 0) {                       // dQ first: it leaves the queries' statistics for dK and dV
        p.splits = n.dq;
        p.part = reinterpret_cast<float*>(p.stat + n.dq_at);
        st = launch_bwd<DP, false, DT>(c, m[0][0], m[0][3], m[1][1], m[1][2], p, norms);
        if (st == OM_OK && n.dq > 1) st = join<DT, false>(c, p, p.dq, p.Sq, p.H);
    }
    if (st == OM_OK && p.Sk > 0) {
        p.splits = n.dkv;
        p.part = reinterpret_cast<float*>(p.stat + n.dkv_at);
        st = launch_bwd<DP, true, DT>(c, m[0][1], m[0][2], m[1][0], m[1][3], p, p.Sq > 0);
        if (st == OM_OK && n.dkv > 1) st = join<DT, false>(c, p, p.dk, p.Sk, p.Hkv, &p.dv);
    }
    return st;
}

}  // namespace attn
}  // namespace omb

using namespace omb;

extern "C" long long omCudaAttentionWorkspaceBytes(int nBatch, int nHeads, int nKvHeads, int nSq,
                                                   int nSk, int nHeadDim, int bBackward) {
    const int st = attn::check_sizes(nBatch, nHeads, nKvHeads, nSq, nSk, nHeadDim);
    if (st != OM_OK) return st;
    const attn::Plan a = attn::plan(nBatch, nHeads, nKvHeads, nSq, nSk, nHeadDim, false);
    const attn::Plan b = attn::plan(nBatch, nHeads, nKvHeads, nSq, nSk, nHeadDim, true);
    return bBackward ? (a.bwd_bytes > b.bwd_bytes ? a.bwd_bytes : b.bwd_bytes)
                     : (a.fwd_bytes > b.fwd_bytes ? a.fwd_bytes : b.fwd_bytes);
}

extern "C" int omCudaAttention(const void* pQ, const void* pK, const void* pV, void* pOut,
                               float* pLse, const long long* pStrides, const int* pQLens,
                               const int* pKvLens, void* pWorkspace, int nBatch, int nHeads,
                               int nKvHeads, int nSq, int nSk, int nHeadDim, float fScale,
                               int bCausal, int nDtype) {
    OMB_CTX_OR_FAIL(c);
    const int st = attn::check_sizes(nBatch, nHeads, nKvHeads, nSq, nSk, nHeadDim);
    if (st != OM_OK) return st;
    if (nDtype != OM_DTYPE_BF16 && nDtype != OM_DTYPE_F16) return OM_ERR_UNSUPPORTED;
    if (!(fabsf(fScale) < INFINITY)) return OM_ERR_INVALID;
    attn::Params p = {};
    if (!pStrides || !attn::view(&p.q, pQ, pStrides, nBatch, nSq, nHeads) ||
        !attn::view(&p.k, pK, pStrides + 3, nBatch, nSk, nKvHeads) ||
        !attn::view(&p.v, pV, pStrides + 6, nBatch, nSk, nKvHeads) ||
        !attn::view(&p.o, pOut, pStrides + 9, nBatch, nSq, nHeads))
        return OM_ERR_INVALID;
    if (nBatch == 0 || nSq == 0) return OM_OK;
    p.lse = pLse; p.qlens = pQLens; p.kvlens = pKvLens;
    p.B = nBatch; p.H = nHeads; p.Hkv = nKvHeads; p.Sq = nSq; p.Sk = nSk; p.D = nHeadDim;
    p.causal = bCausal != 0; p.err = c->err_word;
    attn::set_scale(&p, fScale);
    return nDtype == OM_DTYPE_BF16 ? attn::forward<OM_DTYPE_BF16>(c, p, pWorkspace)
                                    : attn::forward<OM_DTYPE_F16>(c, p, pWorkspace);
}

extern "C" int omCudaAttentionBackward(const void* pGradOut, const void* pQ, const void* pK,
                                       const void* pV, const void* pOut, const float* pLse,
                                       void* pGradQ, void* pGradK, void* pGradV,
                                       const long long* pStrides, const int* pQLens,
                                       const int* pKvLens, void* pWorkspace, int nBatch,
                                       int nHeads, int nKvHeads, int nSq, int nSk, int nHeadDim,
                                       float fScale, int bCausal, int nDtype) {
    OMB_CTX_OR_FAIL(c);
    const int st = attn::check_sizes(nBatch, nHeads, nKvHeads, nSq, nSk, nHeadDim);
    if (st != OM_OK) return st;
    if (nDtype != OM_DTYPE_BF16 && nDtype != OM_DTYPE_F16) return OM_ERR_UNSUPPORTED;
    if (!(fabsf(fScale) < INFINITY)) return OM_ERR_INVALID;
    if (fabsf(fScale) < 0x1p-20f) return OM_ERR_UNSUPPORTED;    // log(keys) / |scale| nears the parts' range
    attn::Params p = {};
    if (!pStrides || !attn::view(&p.q, pQ, pStrides, nBatch, nSq, nHeads) ||
        !attn::view(&p.k, pK, pStrides + 3, nBatch, nSk, nKvHeads) ||
        !attn::view(&p.v, pV, pStrides + 6, nBatch, nSk, nKvHeads) ||
        !attn::view(&p.o, pOut, pStrides + 9, nBatch, nSq, nHeads) ||
        !attn::view(&p.dout, pGradOut, pStrides + 12, nBatch, nSq, nHeads) ||
        !attn::view(&p.dq, pGradQ, pStrides + 15, nBatch, nSq, nHeads) ||
        !attn::view(&p.dk, pGradK, pStrides + 18, nBatch, nSk, nKvHeads) ||
        !attn::view(&p.dv, pGradV, pStrides + 21, nBatch, nSk, nKvHeads))
        return OM_ERR_INVALID;
    if (nBatch == 0) return OM_OK;
    if (nSq > 0 && (!pLse || !pWorkspace || reinterpret_cast<uintptr_t>(pWorkspace) % 16))
        return OM_ERR_INVALID;
    p.lse = const_cast<float*>(pLse); p.stat = static_cast<uint8_t*>(pWorkspace);
    p.qlens = pQLens; p.kvlens = pKvLens;
    p.B = nBatch; p.H = nHeads; p.Hkv = nKvHeads; p.Sq = nSq; p.Sk = nSk; p.D = nHeadDim;
    p.causal = bCausal != 0; p.err = c->err_word;
    attn::set_scale(&p, fScale);
    if (nHeadDim <= 64)
        return nDtype == OM_DTYPE_BF16 ? attn::backward<64, OM_DTYPE_BF16>(c, p) : attn::backward<64, OM_DTYPE_F16>(c, p);
    return nDtype == OM_DTYPE_BF16 ? attn::backward<128, OM_DTYPE_BF16>(c, p) : attn::backward<128, OM_DTYPE_F16>(c, p);
}
