// Attention and its backward, which recomputes the probabilities from the saved log-sum-exp.
#include "om_common.cuh"
#include "om_tc_ptx.cuh"

namespace omb {
namespace attn {

using namespace omb::tc;

struct View {          // a [batch, token, head, D] tensor: element strides, D contiguous
    void* p;
    long long sb, st, sh;
};
struct Params {
    View q, k, v, o, dout, dq, dk, dv;
    float* lse;        // [B, H, Sq]
    float* delta;      // [B, H, Sq], the row sums of dO o O
    const int *qlens, *kvlens;
    int B, H, Hkv, Sq, Sk, D, causal;
    float scale;
    float scale2;      // |scale| * log2(e), not 0 (masked scores stay minus infinity)
    bool neg;          // scale < 0: the score products negate Q
    unsigned int* err;
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
template <int DT>
__device__ float dot(const typename Half16<DT>::T* a, const typename Half16<DT>::T* b, int D) {
    float s = 0.f;
    for (int d = 0; d < D; ++d) s += Half16<DT>::to_f(a[d]) * Half16<DT>::to_f(b[d]);
    return s;
}
__device__ float block_reduce(float v, float* sh, bool is_max) {
    for (int o = 16; o; o >>= 1) {
        const float u = __shfl_xor_sync(~0u, v, o);
        v = is_max ? fmaxf(v, u) : v + u;
    }
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
    __syncthreads();
    v = sh[0];
    for (int w = 1; w < (int)blockDim.x / 32; ++w) v = is_max ? fmaxf(v, sh[w]) : v + sh[w];
    return v;
}

// ---------------------------------------------------------------- tcgen05 pieces
// D[tmem] (+)= A[tmem] * B[smem]: A holds 16-bit pairs, one row per lane, K along the columns.
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc,
                                          uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate));
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
// K-major operand (rows = M or N, K = the head dimension), 16 columns at step k.
__device__ __forceinline__ uint64_t desc_k(uint32_t tile, int k) {
    return smem_desc(tile + (k / 4) * PANEL + (k % 4) * 32, 16, 1024, LAYOUT_SW128);
}
// MN-major operand (rows = K, N = the head dimension), 16 rows at step k.
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, int k) {
    return smem_desc(tile + k * 2048, PANEL, 1024, LAYOUT_SW128);
}
template <int DP>
__device__ __forceinline__ void load_tile(uint32_t dst_off, uint8_t* smem, const CUtensorMap* map,
                                          uint64_t* bar, int t0, int h, int b) {
#pragma unroll
    for (int c = 0; c < DP / 64; ++c)
        tma_load_4d(smem + dst_off + c * PANEL, map, bar, c * 64, t0, h, b);
}
// Rows [first, 128) of a tile become zeros: what lies past a sequence's length must not reach a
// product, since 0 * NaN is NaN. One thread per row.
template <int DP>
__device__ __forceinline__ void zero_tail(uint8_t* tile, int first, int row) {
    if (row >= first) {
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                reinterpret_cast<uint4*>(tile + c * PANEL + row * 128)[i] = make_uint4(0, 0, 0, 0);
    }
    fence_async_smem();
}

// ---------------------------------------------------------------- forward
// One CTA: NT tiles of 128 queries of one (batch, head), over the key blocks of 128. A softmax
// warpgroup per tile (thread = query row), a TMA warp and an MMA warp. Per tile and block:
//   S = Q K^T (TMEM, fp32) -> running maximum, P = exp(S - m), row sums -> P (TMEM, 16-bit, over
//   S's columns) -> O += P V (TMEM, fp32).
// O is rescaled only when a row's maximum has grown by more than 2^8 since its last reference
// maximum: P stays below 2^8, in range of both types, and the factor cancels in O / l.
// TMEM: S_t at t * 128 columns, O_t behind the S tiles.
template <int DP, int NT>
struct FwdCfg {
    static constexpr int TILE = DP / 64 * PANEL;
    static constexpr int SLOTS = NT == 2 ? (DP == 128 ? 4 : 8) : (DP == 128 ? 2 : 5);
    static constexpr int SMEM = (NT + SLOTS) * TILE + 1024 + 1024;
    static constexpr int THREADS = NT * 128 + 64;
    static constexpr int TMEM_COLS = NT * 256;
    static constexpr int O_COL = NT * 128, O_STEP = 128;
};
enum : unsigned int { ERR_LOAD = ERRBIT_TC_PRODUCER, ERR_MMA = ERRBIT_TC_MMA,
                      ERR_MATH = ERRBIT_TC_EPILOGUE, ERR_DRAIN = ERRBIT_TC_DRAIN };

template <int DP, int NT, int DT>
__global__ void __launch_bounds__(NT * 128 + 64, NT == 1 ? 2 : 1)
attn_fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                const __grid_constant__ CUtensorMap mv, const Params p) {
    using Cf = FwdCfg<DP, NT>;
    using H16 = Half16<DT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (NT + Cf::SLOTS) * Cf::TILE);
    uint64_t* q_full = bars;
    uint64_t* o_full = bars + 1;
    uint64_t* drain = bars + 2;
    uint64_t* s_full = bars + 3;
    uint64_t* p_full = s_full + NT;
    uint64_t* full = p_full + NT;
    uint64_t* empty = full + Cf::SLOTS;
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(empty + Cf::SLOTS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    constexpr int W_LOAD = NT * 4, W_MMA = NT * 4 + 1;
    const int h = blockIdx.y % p.H, b = blockIdx.y / p.H, hk = h / (p.H / p.Hkv);
    // the longest rows of a causal mask first
    const int q0 = (p.causal ? gridDim.x - 1 - blockIdx.x : blockIdx.x) * (NT * 128);
    const int ql = len_of(p.qlens, b, p.Sq), kl = len_of(p.kvlens, b, p.Sk);
    int end = q0 < ql ? kl : 0;
    if (p.causal) end = min(end, min(q0 + NT * 128, ql) - 1 + kl - ql + 1);
    const int nblk = end > 0 ? (end + 127) / 128 : 0;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(o_full, 1);
        mbar_init(drain, 1);
        for (int t = 0; t < NT; ++t) { mbar_init(s_full + t, 1); mbar_init(p_full + t, 128); }
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
    const uint32_t tmem = *tmem_holder;
    const uint32_t kv_base = smem_u32(smem) + NT * Cf::TILE;
    unsigned int err = 0;

    if (warp == W_LOAD) {
        if (lane == 0 && nblk > 0) {
            mbar_expect_tx(q_full, NT * Cf::TILE);
            for (int t = 0; t < NT; ++t) load_tile<DP>(t * Cf::TILE, smem, &mq, q_full, q0 + t * 128, h, b);
            int i = 0;
            for (; i < 2 * nblk; ++i) {   // K_0, V_0, K_1, V_1, ...
                const int slot = i % Cf::SLOTS;
                if (!mbar_wait(empty + slot, ((i / Cf::SLOTS) & 1) ^ 1, abort_flag)) { err = ERR_LOAD; break; }
                mbar_expect_tx(full + slot, Cf::TILE);
                load_tile<DP>((NT + slot) * Cf::TILE, smem, i & 1 ? &mv : &mk, full + slot, (i / 2) * 128, hk, b);
            }
            if (err || *abort_flag) {     // every load issued has to land before the CTA ends
                *abort_flag = 1;
                if (!mbar_wait_drain(q_full, 0)) err |= ERR_DRAIN;
                for (int j = max(0, i - Cf::SLOTS); j < i; ++j)
                    if (!mbar_wait_drain(full + j % Cf::SLOTS, (j / Cf::SLOTS) & 1)) err |= ERR_DRAIN;
            }
        }
    } else if (warp == W_MMA) {
        if (lane == 0 && nblk > 0) {
            const int ks = (p.D + 15) / 16;
            const uint32_t id_s = idesc_f16(DT == OM_DTYPE_F16, 128, false, p.neg);
            const uint32_t id_o = idesc_f16(DT == OM_DTYPE_F16, ks * 16, true, false);
            const uint32_t q_tile = smem_u32(smem);
            auto qk = [&](int t, int i) {
                const uint32_t kt = kv_base + (i % Cf::SLOTS) * Cf::TILE;
                for (int k = 0; k < ks; ++k)
                    tc_mma(tmem + t * 128, desc_k(q_tile + t * Cf::TILE, k), desc_k(kt, k), id_s, k > 0);
                tc_commit(s_full + t);
            };
            auto wait_kv = [&](int i) { return mbar_wait(full + i % Cf::SLOTS, (i / Cf::SLOTS) & 1, abort_flag); };
            bool ok = mbar_wait(q_full, 0, abort_flag) && wait_kv(0);
            if (ok) {
                tc_fence_after();
                for (int t = 0; t < NT; ++t) qk(t, 0);
                tc_commit(empty + 0);
            }
            for (int j = 0; ok && j < nblk; ++j) {
                const bool more = j + 1 < nblk;
                ok = wait_kv(2 * j + 1) && (!more || wait_kv(2 * j + 2));
                const uint32_t vt = kv_base + ((2 * j + 1) % Cf::SLOTS) * Cf::TILE;
                for (int t = 0; ok && t < NT; ++t) {
                    ok = mbar_wait(p_full + t, j & 1, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
                    for (int k = 0; k < 8; ++k)
                        tc_mma_ts(tmem + Cf::O_COL + t * Cf::O_STEP, tmem + t * 128 + k * 8, desc_mn(vt, k), id_o,
                                  j > 0 || k > 0);
                    if (more) qk(t, 2 * j + 2);
                }
                if (!ok) break;
                tc_commit(empty + (2 * j + 1) % Cf::SLOTS);
                tc_commit(more ? empty + (2 * j + 2) % Cf::SLOTS : o_full);
            }
            if (!ok) {                    // no MMA may run on when the CTA ends
                *abort_flag = 1;
                err = ERR_MMA;
                tc_commit(drain);
                if (!mbar_wait_drain(drain, 0)) err |= ERR_DRAIN;
            }
        }
        __syncwarp();
    } else {
        const int t = warp / 4, row = (warp % 4) * 32 + lane;
        const int i = q0 + t * 128 + row;
        const uint32_t s_addr = tmem + t * 128 + ((uint32_t)(warp % 4) << 21);
        const uint32_t o_addr = tmem + Cf::O_COL + t * Cf::O_STEP + ((uint32_t)(warp % 4) << 21);
        int row_end = i < ql ? kl : 0;
        if (p.causal) row_end = min(row_end, i + kl - ql + 1);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < nblk; ++j) {
            ok = __all_sync(~0u, mbar_wait(s_full + t, j & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            uint32_t sv[128];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32_issue(s_addr + c * 32, sv + c * 32);
            tmem_ld_wait<128>(sv);
            float* s = reinterpret_cast<float*>(sv);
            const int seen = row_end - j * 128;      // columns of this block that the row sees
            if (__any_sync(~0u, seen < 128)) {
#pragma unroll
                for (int c = 0; c < 128; ++c) s[c] = c < seen ? s[c] : -INFINITY;
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int c = 4; c < 128; ++c) mx[c % 4] = fmaxf(mx[c % 4], s[c]);
            const float m_new = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), m);
            if (j == 0) {
                m = m_new;
            } else if (__any_sync(~0u, (m_new - m) * p.scale2 > 8.f)) {
                // S_j is complete, so every product issued before it is: O may be changed
                const float f = m == -INFINITY ? 0.f : ex2((m - m_new) * p.scale2);
                l *= f;
                m = m_new;
                for (int c = 0; c < p.D; c += 32) {
                    uint32_t o[32];
                    tmem_ld32_issue(o_addr + c, o);
                    tmem_ld_wait<32>(o);
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                    tmem_st32(o_addr + c, o);
                }
                tmem_st_wait();
            }
            const float sub = m == -INFINITY ? 0.f : -m * p.scale2;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t w[16];
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float a = ex2(fmaf(s[c * 32 + 2 * x], p.scale2, sub));
                    const float d = ex2(fmaf(s[c * 32 + 2 * x + 1], p.scale2, sub));
                    sum[x % 2 * 2] += a;
                    sum[x % 2 * 2 + 1] += d;
                    w[x] = pack16<DT>(a, d);
                }
                tmem_st16(s_addr + c * 16, w);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            // keys past the sequence's length may hold anything
            if (t == 0 && j == nblk - 1 && kl - j * 128 < 128) {
                const int iv = 2 * j + 1;
                ok = __all_sync(~0u, mbar_wait(full + iv % Cf::SLOTS, (iv / Cf::SLOTS) & 1, abort_flag));
                if (!ok) break;
                zero_tail<DP>(smem + (NT + iv % Cf::SLOTS) * Cf::TILE, kl - j * 128, row);
            }
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(p_full + t);
        }
        if (ok && nblk > 0) ok = __all_sync(~0u, mbar_wait(o_full, 0, abort_flag));
        if (!ok) {
            *abort_flag = 1;
            err = ERR_MATH;
        } else {
            tc_fence_after();
            const float inv = l > 0.f ? 1.f / l : 0.f;
            auto* out = i < p.Sq ? row_out<DT>(p.o, b, i, h) : nullptr;
            for (int c = 0; c < p.D; c += 32) {
                uint32_t o[32];
                if (nblk > 0) {
                    tmem_ld32_issue(o_addr + c, o);
                    tmem_ld_wait<32>(o);
                }
                const int n8 = min(32, p.D - c) / 8;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t w[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        w[y] = nblk > 0 ? pack16<DT>(__uint_as_float(o[x * 8 + 2 * y]) * inv,
                                                     __uint_as_float(o[x * 8 + 2 * y + 1]) * inv)
                                        : 0u;
                    if (out && x < n8)
                        reinterpret_cast<uint4*>(out + c)[x] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            if (p.lse && i < p.Sq)
                p.lse[((long long)b * p.H + h) * p.Sq + i] =
                    l > 0.f ? (m * p.scale2 + log2f(l)) * 0.6931471805599453f : -INFINITY;
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

template <int DT>
__global__ void __launch_bounds__(128) attn_dq_kernel(const Params p) {
    using H16 = Half16<DT>;
    __shared__ float sp[128];
    const int i = blockIdx.x, h = blockIdx.y % p.H, b = blockIdx.y / p.H, t = threadIdx.x;
    const int hk = h / (p.H / p.Hkv);
    const int ql = len_of(p.qlens, b, p.Sq), kl = len_of(p.kvlens, b, p.Sk);
    int end = i < ql ? kl : 0;
    if (p.causal) end = min(end, i + kl - ql + 1);
    const long long at = ((long long)b * p.H + h) * p.Sq + i;
    const float lse = p.lse[at];
    const float delta = end > 0 ? dot<DT>(row<DT>(p.dout, b, i, h), row<DT>(p.o, b, i, h), p.D) : 0.f;
    if (t == 0) p.delta[at] = delta;
    float acc = 0.f;
    for (int j0 = 0; j0 < end; j0 += 128) {
        const int j = j0 + t;
        float ds = 0.f;
        if (j < end) {
            const float w = expf(dot<DT>(row<DT>(p.q, b, i, h), row<DT>(p.k, b, j, hk), p.D) * p.scale - lse);
            ds = w * (dot<DT>(row<DT>(p.dout, b, i, h), row<DT>(p.v, b, j, hk), p.D) - delta) * p.scale;
        }
        __syncthreads();
        sp[t] = ds;
        __syncthreads();
        if (t < p.D)
            for (int jj = 0; jj < min(128, end - j0); ++jj)
                acc += sp[jj] * H16::to_f(row<DT>(p.k, b, j0 + jj, hk)[t]);
    }
    if (t < p.D) row_out<DT>(p.dq, b, i, h)[t] = H16::from_f(acc);
}

// One block per (batch, key/value head, key), after attn_dq_kernel has left delta.
template <int DT>
__global__ void __launch_bounds__(128) attn_dkv_kernel(const Params p) {
    using H16 = Half16<DT>;
    __shared__ float sp[128], sd[128];
    const int j = blockIdx.x, hk = blockIdx.y % p.Hkv, b = blockIdx.y / p.Hkv, t = threadIdx.x;
    const int ql = len_of(p.qlens, b, p.Sq), kl = len_of(p.kvlens, b, p.Sk);
    const int first = p.causal ? max(0, j - (kl - ql)) : 0;
    float dk = 0.f, dv = 0.f;
    if (j < kl)
        for (int h = hk * (p.H / p.Hkv); h < (hk + 1) * (p.H / p.Hkv); ++h)
            for (int i0 = first; i0 < ql; i0 += 128) {
                const int i = i0 + t;
                float w = 0.f, ds = 0.f;
                if (i < ql) {
                    const long long at = ((long long)b * p.H + h) * p.Sq + i;
                    w = expf(dot<DT>(row<DT>(p.q, b, i, h), row<DT>(p.k, b, j, hk), p.D) * p.scale - p.lse[at]);
                    ds = w * (dot<DT>(row<DT>(p.dout, b, i, h), row<DT>(p.v, b, j, hk), p.D) - p.delta[at]) * p.scale;
                }
                __syncthreads();
                sp[t] = w;
                sd[t] = ds;
                __syncthreads();
                if (t < p.D)
                    for (int ii = 0; ii < min(128, ql - i0); ++ii) {
                        dv += sp[ii] * H16::to_f(row<DT>(p.dout, b, i0 + ii, h)[t]);
                        dk += sd[ii] * H16::to_f(row<DT>(p.q, b, i0 + ii, h)[t]);
                    }
            }
    if (t < p.D) {
        row_out<DT>(p.dk, b, j, hk)[t] = H16::from_f(dk);
        row_out<DT>(p.dv, b, j, hk)[t] = H16::from_f(dv);
    }
}

static int check_sizes(int nBatch, int nHeads, int nKvHeads, int nSq, int nSk, int nHeadDim) {
    if (nBatch < 0 || nHeads <= 0 || nKvHeads <= 0 || nHeads % nKvHeads || nSq < 0 || nSk < 0 ||
        nHeadDim <= 0)
        return OM_ERR_INVALID;
    if (nHeadDim % 8 || nHeadDim > 128 || (long long)nBatch * nHeads > 65535)
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
}

// A tensor map over a [batch, token, head, D] view with boxes of 64 columns x 128 tokens.
// Strides of dimensions of length 1 are replaced by one that the map takes.
static int encode(CUtensorMap* map, const View& v, int nB, int nT, int nH, int D, int dt) {
    PFN_cuTensorMapEncodeTiled_v12000 fn = tc::encode_tiled_fn();
    if (!fn) return OM_ERR_DRIVER;
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)nT, (cuuint64_t)nH, (cuuint64_t)nB};
    cuuint64_t strides[3] = {nT > 1 ? (cuuint64_t)v.st * 2 : 256, nH > 1 ? (cuuint64_t)v.sh * 2 : 256,
                             nB > 1 ? (cuuint64_t)v.sb * 2 : 256};
    cuuint32_t box[4] = {64, 128, 1, 1};
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
        OMB_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cf::SMEM));
        attr_set[c->device] = true;
    }
    CUtensorMap mq = {}, mk = {}, mv = {};
    int st = encode(&mq, p.q, p.B, p.Sq, p.H, p.D, DT);
    if (st == OM_OK && p.Sk > 0) st = encode(&mk, p.k, p.B, p.Sk, p.Hkv, p.D, DT);
    if (st == OM_OK && p.Sk > 0) st = encode(&mv, p.v, p.B, p.Sk, p.Hkv, p.D, DT);
    if (st != OM_OK) return st;
    const dim3 grid((p.Sq + NT * 128 - 1) / (NT * 128), p.B * p.H);
    kern<<<grid, Cf::THREADS, Cf::SMEM, c->compute>>>(mq, mk, mv, p);
    return after_launch(c);
}
template <int DT>
static int forward(DeviceCtx* c, const Params& p) {
    if (p.D <= 64) return p.Sq <= 128 ? launch_fwd<64, 1, DT>(c, p) : launch_fwd<64, 2, DT>(c, p);
    return p.Sq <= 128 ? launch_fwd<128, 1, DT>(c, p) : launch_fwd<128, 2, DT>(c, p);
}

}  // namespace attn
}  // namespace omb

using namespace omb;

extern "C" long long omCudaAttentionWorkspaceBytes(int nBatch, int nHeads, int nKvHeads, int nSq,
                                                   int nSk, int nHeadDim, int bBackward) {
    const int st = attn::check_sizes(nBatch, nHeads, nKvHeads, nSq, nSk, nHeadDim);
    if (st != OM_OK) return st;
    return bBackward ? (long long)nBatch * nHeads * nSq * 4 : 0;
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
    return nDtype == OM_DTYPE_BF16 ? attn::forward<OM_DTYPE_BF16>(c, p) : attn::forward<OM_DTYPE_F16>(c, p);
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
    p.lse = const_cast<float*>(pLse); p.delta = static_cast<float*>(pWorkspace);
    p.qlens = pQLens; p.kvlens = pKvLens;
    p.B = nBatch; p.H = nHeads; p.Hkv = nKvHeads; p.Sq = nSq; p.Sk = nSk; p.D = nHeadDim;
    p.causal = bCausal != 0; p.err = c->err_word;
    attn::set_scale(&p, fScale);
    if (nSq > 0) {
        const dim3 grid(nSq, nBatch * nHeads);
        if (nDtype == OM_DTYPE_BF16)
            attn::attn_dq_kernel<OM_DTYPE_BF16><<<grid, 128, 0, c->compute>>>(p);
        else
            attn::attn_dq_kernel<OM_DTYPE_F16><<<grid, 128, 0, c->compute>>>(p);
        if (after_launch(c) != OM_OK) return OM_ERR_CUDA;
    }
    if (nSk > 0) {
        const dim3 grid(nSk, nBatch * nKvHeads);
        if (nDtype == OM_DTYPE_BF16)
            attn::attn_dkv_kernel<OM_DTYPE_BF16><<<grid, 128, 0, c->compute>>>(p);
        else
            attn::attn_dkv_kernel<OM_DTYPE_F16><<<grid, 128, 0, c->compute>>>(p);
        if (after_launch(c) != OM_OK) return OM_ERR_CUDA;
    }
    return OM_OK;
}
