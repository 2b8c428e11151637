// GroupNorm with its activation on channels-last maps, forward and backward.
//
// z = gamma_c (x - mean) rstd + beta_c, y = act(z), statistics over the HW x C/G values of each
// (sample, group). Backward, with dz = dy act'(z), xh = (x - mean) rstd and t = gamma_c dz:
//   dbeta_c = sum dz, dgamma_c = sum dz xh, dx = rstd (t - mean(t) - xh mean(t xh)),
// where the group means follow from the per-channel sums: mean(t) = sum_c gamma_c A_c / M with
// A_c = sum dz, mean(t xh) = sum_c gamma_c B_c / M with B_c = sum dz xh.
//
// Bound by memory: the floor is one read of each input and one write of the output. A unit is
// one sample's slab of channels (whole groups, at least 64 bytes of a pixel where there are as
// many). Where a unit fits the shared memory of a cluster of up to 8 CTAs, one kernel reads it
// once into shared memory, exchanges the sums over the cluster's distributed shared memory and
// writes the output from there. Larger units take three launches: partial sums per chunk of
// pixels, their combination, and the pass that reads the input again.
// Statistics are fp32 means and centred sums of squares, merged pairwise (Chan, Golub, LeVeque,
// 1979), so a mean far from zero costs no precision; every merge has a fixed order.
#include <cooperative_groups.h>

#include <type_traits>

#include "om_common.cuh"
#include "om_f2.cuh"

namespace omb {
namespace gn {

namespace cg = cooperative_groups;

constexpr int T = 256;                    // threads of every block
constexpr int MAX_VC = 256;               // 8-channel vectors of a pixel that one block covers
constexpr int MAX_CLUSTER = 8;
constexpr int SMEM_MAX = 227 * 1024;
constexpr int KEEP_MAX = SMEM_MAX / 2 - 1024, KEEP_GOOD = SMEM_MAX / 4 - 1024;
constexpr int MAX_GROUPS = 40;            // of a slab: it ends with the first unit of lcm(cpg, 8)
                                          // channels that reaches 32, so below 32 / cpg + 8

template <int DT> struct Elem { using T = float; static constexpr int V16 = 2; };
template <> struct Elem<OM_DTYPE_BF16> { using T = __nv_bfloat16; static constexpr int V16 = 1; };
template <> struct Elem<OM_DTYPE_F16> { using T = __half; static constexpr int V16 = 1; };

// 8 channels of one pixel: V16 16-byte pieces
template <int DT> struct Vec { uint4 q[Elem<DT>::V16]; };

template <int DT>
__device__ __forceinline__ void unpack(const Vec<DT>& v, F2 (&f)[4]) {
    if constexpr (DT == OM_DTYPE_F32) {
        const float* s = reinterpret_cast<const float*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = {s[2 * i], s[2 * i + 1]};
    } else {
        const auto* s = reinterpret_cast<const typename Half16<DT>::T2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 u = Half16<DT>::unpack(s[i]);
            f[i] = {u.x, u.y};
        }
    }
}
template <int DT>
__device__ __forceinline__ Vec<DT> pack(const F2 (&f)[4]) {
    Vec<DT> v;
    if constexpr (DT == OM_DTYPE_F32) {
        float* d = reinterpret_cast<float*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) { d[2 * i] = f[i].x; d[2 * i + 1] = f[i].y; }
    } else {
        auto* d = reinterpret_cast<typename Half16<DT>::T2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = Half16<DT>::pack(f[i].x, f[i].y);
    }
    return v;
}
// channels past nval (stored padding) as zeros, whatever they hold
__device__ __forceinline__ void cut(F2 (&f)[4], int nval) {
    if (nval < 8)
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = {2 * i < nval ? f[i].x : 0.f, 2 * i + 1 < nval ? f[i].y : 0.f};
}
template <int DT>
__device__ __forceinline__ Vec<DT> load(const void* base, long long elem) {
    Vec<DT> v;
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const typename Elem<DT>::T*>(base) + elem);
#pragma unroll
    for (int i = 0; i < Elem<DT>::V16; ++i) v.q[i] = __ldg(s + i);
    return v;
}
template <int DT>
__device__ __forceinline__ void store(void* base, long long elem, const Vec<DT>& v) {
    uint4* d = reinterpret_cast<uint4*>(static_cast<typename Elem<DT>::T*>(base) + elem);
#pragma unroll
    for (int i = 0; i < Elem<DT>::V16; ++i) d[i] = v.q[i];
}
// Slot s of a thread's own shared memory, in planes of T 16-byte pieces (no bank conflicts); the
// copy is asynchronous and only the thread that issued it reads it.
template <int DT>
__device__ __forceinline__ void copy_in(uint4* sm, int s, const void* base, long long elem) {
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const typename Elem<DT>::T*>(base) + elem);
#pragma unroll
    for (int i = 0; i < Elem<DT>::V16; ++i)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         (uint32_t)__cvta_generic_to_shared(sm + (s * Elem<DT>::V16 + i) * T + threadIdx.x)),
                     "l"(src + i) : "memory");
}
template <int DT>
__device__ __forceinline__ Vec<DT> own(const uint4* sm, int s) {
    Vec<DT> v;
#pragma unroll
    for (int i = 0; i < Elem<DT>::V16; ++i) v.q[i] = sm[(s * Elem<DT>::V16 + i) * T + threadIdx.x];
    return v;
}
// sigmoid(z) = 1 / (1 + 2^(-z log2 e)): an overflowing power gives 0
__device__ __forceinline__ F2 sigmoid(F2 z) {
    F2 e = mul2(z, {-1.4426950408889634f, -1.4426950408889634f}), s;
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.y));
    e = add2(e, {1.f, 1.f});
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(e.y));
    return s;
}
template <int ACT>
__device__ __forceinline__ F2 act_fwd(F2 z) {
    if (ACT == OM_ACT_SILU) return mul2(z, sigmoid(z));
    return {apply_act(z.x, ACT), apply_act(z.y, ACT)};
}
// dz = dy * act'(z)
template <int ACT>
__device__ __forceinline__ F2 act_bwd(F2 dy, F2 z) {
    if (ACT == OM_ACT_SILU) {             // s (1 + z (1 - s))
        const F2 s = sigmoid(z), zs = mul2(z, s);
        return mul2(dy, mul2(s, add2(fma2(zs, {-1.f, -1.f}, z), {1.f, 1.f})));
    }
    if (ACT == OM_ACT_RELU) return {z.x > 0.f ? dy.x : 0.f, z.y > 0.f ? dy.y : 0.f};
    if (ACT == OM_ACT_RELU6)
        return {z.x > 0.f && z.x < 6.f ? dy.x : 0.f, z.y > 0.f && z.y < 6.f ? dy.y : 0.f};
    return dy;
}

struct Params {
    const void *x, *dy;
    void* out;
    const float *gamma, *beta;
    float *mean, *rstd;       // [N, G]: written by the forward when given, read by the backward
    float *dgamma, *dbeta;
    float* ws;
    int N, HW, C, Cs, G;
    float eps;
    int cpg;
    int vc;                   // vectors of a slab
    int nslab;
    int cluster;              // CTAs of a unit
    int rows;                 // pixels of a CTA's part
    int iters;                // of them per thread
    int nchunk;               // parts of a sample (three-launch form)
};

// What a thread works on: vector column cv of pixels first, first + step, ... < end
struct Part {
    int n, c0, nval;          // sample, first channel, channels of it that are not padding
    int first, step, end;
    bool active;
    long long base;           // element of (n, pixel 0, c0)
};
__device__ __forceinline__ Part part_of(const Params& p, int n, int slab, int piece) {
    Part t;
    const int cv = threadIdx.x % p.vc, r = threadIdx.x / p.vc;
    t.n = n;
    t.step = T / p.vc;
    t.c0 = (slab * p.vc + cv) * 8;
    t.active = r < t.step && t.c0 < p.Cs;
    t.nval = min(max(p.C - t.c0, 0), 8);
    t.first = piece * p.rows + r;
    t.end = t.active ? min((piece + 1) * p.rows, p.HW) : 0;
    t.base = (long long)n * p.HW * p.Cs + t.c0;
    return t;
}
__device__ __forceinline__ long long at(const Params& p, const Part& t, int pixel) {
    return t.base + (long long)pixel * p.Cs;
}

// NV pairs of values of every thread, added over the threads of the same vector column: the
// results land in sums[2][vc * NV]. red: T * 2 * NV floats. A fixed order; ends with a barrier.
template <int NV>
__device__ void reduce_columns(const Params& p, float (&a)[NV], float (&b)[NV], float* red, float* sums) {
    const int R = T / p.vc, cv = threadIdx.x % p.vc, r = threadIdx.x / p.vc;
    int rows = R, slot = threadIdx.x;
    bool write = r < R;
    if (p.vc <= 16 && (p.vc & (p.vc - 1)) == 0) {   // a warp holds 32 / vc whole rows
        for (int o = 16; o >= p.vc; o >>= 1)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                a[i] += __shfl_xor_sync(~0u, a[i], o);
                b[i] += __shfl_xor_sync(~0u, b[i], o);
            }
        rows = T / 32;
        slot = threadIdx.x / 32 * p.vc + cv;
        write = threadIdx.x % 32 < p.vc;
    }
    if (write)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            red[slot * 2 * NV + i] = a[i];
            red[slot * 2 * NV + NV + i] = b[i];
        }
    __syncthreads();
    for (int c = threadIdx.x; c < p.vc * 2 * NV; c += T) {   // c: vector, then a or b, then value
        float s = 0.f;
        for (int k = 0; k < rows; ++k) s += red[k * p.vc * 2 * NV + c];
        sums[c % (2 * NV) / NV * p.vc * NV + c / (2 * NV) * NV + c % NV] = s;
    }
    __syncthreads();
}

// Per-thread running statistics of the GV entries of a vector, 8 / GV channels each: batches of B
// pixels are centred on their own mean and merged.
template <int GV>
struct Stats {
    float mean[GV], m2[GV], n;
    __device__ __forceinline__ void clear() {
        n = 0.f;
#pragma unroll
        for (int g = 0; g < GV; ++g) mean[g] = m2[g] = 0.f;
    }
    template <int B>
    __device__ __forceinline__ void add(const F2 (&v)[B][4]) {
        constexpr float cnt = B * (8 / GV);
        const float w = __fdividef(cnt, n + cnt), k = n * w;
        auto merge = [&](int g, float m, float q) {
            const float d = m - mean[g];
            mean[g] = fmaf(d, w, mean[g]);
            m2[g] += fmaf(d * d, k, q);
        };
        if constexpr (GV == 8) {              // both halves of a pair are entries of their own
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                F2 s = v[0][i], q = {0.f, 0.f};
#pragma unroll
                for (int j = 1; j < B; ++j) s = add2(s, v[j][i]);
                const F2 m = mul2(s, {1.f / cnt, 1.f / cnt}), nm = {-m.x, -m.y};
#pragma unroll
                for (int j = 0; j < B; ++j) {
                    const F2 e = add2(v[j][i], nm);
                    q = fma2(e, e, q);
                }
                merge(2 * i, m.x, q.x);
                merge(2 * i + 1, m.y, q.y);
            }
        } else {
            constexpr int PAIRS = 4 / GV;
#pragma unroll
            for (int g = 0; g < GV; ++g) {
                F2 s = {0.f, 0.f}, q = {0.f, 0.f};
#pragma unroll
                for (int j = 0; j < B; ++j)
#pragma unroll
                    for (int i = 0; i < PAIRS; ++i) s = add2(s, v[j][g * PAIRS + i]);
                const float m = (s.x + s.y) * (1.f / cnt);
#pragma unroll
                for (int j = 0; j < B; ++j)
#pragma unroll
                    for (int i = 0; i < PAIRS; ++i) {
                        const F2 e = add2(v[j][g * PAIRS + i], {-m, -m});
                        q = fma2(e, e, q);
                    }
                merge(g, m, q.x + q.y);
            }
        }
        n += cnt;
    }
};
// The mean and centred sum of squares of each entry over the block's pixels (count values of an
// entry), into sums[0][e], sums[1][e].
template <int GV>
__device__ void block_stats(const Params& p, const Stats<GV>& st, float count, float* red, float* sums) {
    float a[GV], b[GV], m[GV];
#pragma unroll
    for (int i = 0; i < GV; ++i) { a[i] = st.mean[i] * st.n; b[i] = 0.f; }
    reduce_columns<GV>(p, a, b, red, sums);
    const int cv = threadIdx.x % p.vc;
    const float inv = 1.f / count;
#pragma unroll
    for (int i = 0; i < GV; ++i) {
        m[i] = sums[cv * GV + i] * inv;
        const float d = st.mean[i] - m[i];
        a[i] = 0.f;
        b[i] = st.n > 0.f ? fmaf(st.n * d, d, st.m2[i]) : 0.f;
    }
    __syncthreads();
    reduce_columns<GV>(p, a, b, red, sums);
    if (threadIdx.x < p.vc)
#pragma unroll
        for (int i = 0; i < GV; ++i) sums[threadIdx.x * GV + i] = m[i];
    __syncthreads();
}

// z = (x - mean) scale + shift of a thread's 8 channels; with 16-bit inputs the mean is folded into
// the shift (its rounding, 2^-24 of mean * scale, is that of the mean itself). Padding: 0. Not for ReLU
// and ReLU6, whose backward has to see the sign that the forward saw: see Normal.
template <int DT>
struct Affine {
    F2 minus_mean[DT == OM_DTYPE_F32 ? 4 : 1], scale[4], shift[4];
};
__device__ __forceinline__ float& half_of(F2* f, int i) { return i % 2 ? f[i / 2].y : f[i / 2].x; }
template <int DT, class MeanOf, class RstdOf>
__device__ __forceinline__ void affine_of(const Params& p, const Part& t, Affine<DT>& f, MeanOf mean_of, RstdOf rstd_of) {
    int g = t.c0 / p.cpg, left = p.cpg - (t.c0 - g * p.cpg);     // group of the channel, channels left in it
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float m = 0.f, scale = 0.f, shift = 0.f;
        if (i < t.nval) {
            const int c = t.c0 + i;
            m = mean_of(g);
            scale = rstd_of(g) * (p.gamma ? p.gamma[c] : 1.f);
            shift = p.beta ? p.beta[c] : 0.f;
            if (DT != OM_DTYPE_F32) shift = fmaf(-m, scale, shift);
        }
        half_of(f.scale, i) = scale;
        half_of(f.shift, i) = shift;
        if (DT == OM_DTYPE_F32) half_of(f.minus_mean, i) = -m;
        if (--left == 0) { ++g; left = p.cpg; }
    }
}
template <int DT, int ACT>
__device__ __forceinline__ Vec<DT> apply(const Vec<DT>& v, const Affine<DT>& f, int nval) {
    F2 x[4];
    unpack<DT>(v, x);
    cut(x, nval);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        x[i] = act_fwd<ACT>(fma2(DT == OM_DTYPE_F32 ? add2(x[i], f.minus_mean[DT == OM_DTYPE_F32 ? i : 0]) : x[i],
                                 f.scale[i], f.shift[i]));
    return pack<DT>(x);
}

// The coefficients of z = ((x - mean) rstd) gamma + beta of a thread's 8 channels; statistics once per
// entry of GV (channel i belongs to entry i * GV / 8).
template <int GV>
struct Normal {
    float minus_mean[GV], rstd[GV];
    F2 gamma[4], beta[4];
};
// the pair i of a vector from values per entry
template <int GV>
__device__ __forceinline__ F2 pair_of(const float (&v)[GV], int i) {
    return {v[2 * i * GV / 8], v[(2 * i + 1) * GV / 8]};
}
template <int GV, class MeanOf, class RstdOf>
__device__ __forceinline__ void normal_of(const Params& p, const Part& t, Normal<GV>& f, MeanOf mean_of, RstdOf rstd_of) {
    int g = t.c0 / p.cpg, left = p.cpg - (t.c0 - g * p.cpg);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool in = i < t.nval;
        if (i % (8 / GV) == 0) {
            f.minus_mean[i * GV / 8] = in ? -mean_of(g) : 0.f;
            f.rstd[i * GV / 8] = in ? rstd_of(g) : 0.f;
        }
        half_of(f.gamma, i) = !in ? 0.f : p.gamma ? p.gamma[t.c0 + i] : 1.f;
        half_of(f.beta, i) = in && p.beta ? p.beta[t.c0 + i] : 0.f;
        if (--left == 0) { ++g; left = p.cpg; }
    }
}
template <int ACT> constexpr bool HAS_KINK = ACT == OM_ACT_RELU || ACT == OM_ACT_RELU6;
template <int GV>
__device__ __forceinline__ F2 normalised(F2 x, const Normal<GV>& f, int i) {
    return mul2(add2(x, pair_of<GV>(f.minus_mean, i)), pair_of<GV>(f.rstd, i));
}
// z of the pair i. Where its sign decides, product and sum are rounded apart, as the formula reads, in
// both passes: fused (as the paired instructions can be), a z that rounds to 0 came out next to 0 and
// let its gradient through; rounded otherwise in the forward than in the backward, constant maps gave
// outputs above 0 that no gradient came back through
template <int ACT, int GV>
__device__ __forceinline__ F2 pre_activation(F2 xh, const Normal<GV>& f, int i) {
    if (!HAS_KINK<ACT>) return fma2(xh, f.gamma[i], f.beta[i]);
    return {__fadd_rn(__fmul_rn(xh.x, f.gamma[i].x), f.beta[i].x), __fadd_rn(__fmul_rn(xh.y, f.gamma[i].y), f.beta[i].y)};
}
template <int DT, int ACT, int GV>
__device__ __forceinline__ Vec<DT> apply(const Vec<DT>& v, const Normal<GV>& f, int nval) {
    F2 x[4];
    unpack<DT>(v, x);
    cut(x, nval);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = act_fwd<ACT>(pre_activation<ACT, GV>(normalised<GV>(x[i], f, i), f, i));
    return pack<DT>(x);
}
// the forward's coefficients and what it does with them
template <int DT, int ACT, int GV> struct Forward {
    Affine<DT> f;
    template <class M, class R> __device__ __forceinline__ Forward(const Params& p, const Part& t, M mean_of, R rstd_of) {
        affine_of<DT>(p, t, f, mean_of, rstd_of);
    }
    __device__ __forceinline__ Vec<DT> operator()(const Vec<DT>& v, int nval) const { return apply<DT, ACT>(v, f, nval); }
};
template <int DT, int ACT, int GV> struct ForwardKink {
    Normal<GV> f;
    template <class M, class R> __device__ __forceinline__ ForwardKink(const Params& p, const Part& t, M mean_of, R rstd_of) {
        normal_of<GV>(p, t, f, mean_of, rstd_of);
    }
    __device__ __forceinline__ Vec<DT> operator()(const Vec<DT>& v, int nval) const { return apply<DT, ACT, GV>(v, f, nval); }
};
template <int DT, int ACT, int GV>
using ForwardOf = std::conditional_t<HAS_KINK<ACT>, ForwardKink<DT, ACT, GV>, Forward<DT, ACT, GV>>;

// ---------------------------------------------------------------- one launch, unit in a cluster
// GV: entries of a vector whose statistics are kept apart: 1 where a vector lies within a group
// (channels per group a multiple of 8), 2 with 4 channels a group, else 8.
template <int DT, int ACT, int GV>
__global__ void __launch_bounds__(T, 4) gn_fwd_unit_kernel(const Params p) {
    extern __shared__ uint4 sm[];
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), unit = blockIdx.x / p.cluster;
    const int n = unit / p.nslab, slab = unit - n * p.nslab;
    const Part t = part_of(p, n, slab, rank);
    float* red = reinterpret_cast<float*>(sm + p.iters * Elem<DT>::V16 * T);
    float* sums = red + T * 2 * GV;
    float* group = sums + p.vc * 2 * GV;        // mean and m2 of each group over the CTA's pixels
    float* total = group + 2 * MAX_GROUPS;  // mean and rstd over the unit
    const long long step = (long long)t.step * p.Cs;
    const int mine_rows = t.first < t.end ? (t.end - t.first + t.step - 1) / t.step : 0;
    const int half = mine_rows / 2 & ~3;    // statistics of the first half while the second arrives
    {
        long long e = at(p, t, t.first);
        for (int s = 0; s < half; ++s, e += step) copy_in<DT>(sm, s, p.x, e);
        asm volatile("cp.async.commit_group;" ::: "memory");
        for (int s = half; s < mine_rows; ++s, e += step) copy_in<DT>(sm, s, p.x, e);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    Stats<GV> st;
    st.clear();
    auto take = [&](int s, int end) {
        for (; s + 3 < end; s += 4) {
            F2 v[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) unpack<DT>(own<DT>(sm, s + j), v[j]);
            st.template add<4>(v);
        }
        for (; s < end; ++s) {
            F2 v[1][4];
            unpack<DT>(own<DT>(sm, s), v[0]);
            st.template add<1>(v);
        }
    };
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    take(0, half);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    take(half, mine_rows);
    constexpr float PER = 8 / GV;
    const int c_lo = slab * p.vc * 8, g_lo = c_lo / p.cpg;
    const int ng = max(0, min(p.C, c_lo + p.vc * 8) - c_lo) / p.cpg;     // whole groups of the slab
    const int epg = p.cpg * GV / 8;                                      // entries of a group
    const float mine = PER * (float)max(0, min((rank + 1) * p.rows, p.HW) - rank * p.rows);
    block_stats<GV>(p, st, fmaxf(mine, 1.f), red, sums);
    for (int g = threadIdx.x; g < ng; g += T) {
        float m = 0.f, q = 0.f;
        for (int e = 0; e < epg; ++e) m += sums[g * epg + e];
        m /= (float)epg;
        for (int e = 0; e < epg; ++e) {
            const float d = sums[g * epg + e] - m;
            q += sums[p.vc * GV + g * epg + e] + mine * d * d;
        }
        group[2 * g] = m;
        group[2 * g + 1] = q;
    }
    if (p.cluster > 1) cl.sync(); else __syncthreads();
    for (int g = threadIdx.x; g < ng; g += T) {
        // all CTAs' values are on their way before the first is used (one by one their latencies
        // added up to a sixth of the kernel)
        float mk[MAX_CLUSTER], qk[MAX_CLUSTER], m = 0.f, q = 0.f;
#pragma unroll
        for (int k = 0; k < MAX_CLUSTER; ++k)
            if (k < p.cluster) {
                const float* o = cl.map_shared_rank(group, k);
                mk[k] = o[2 * g];
                qk[k] = o[2 * g + 1];
            }
        auto pixels = [&](int k) { return (float)max(0, min((k + 1) * p.rows, p.HW) - k * p.rows); };
#pragma unroll
        for (int k = 0; k < MAX_CLUSTER; ++k)
            if (k < p.cluster) m = fmaf(pixels(k), mk[k], m);
        m /= (float)p.HW;
#pragma unroll
        for (int k = 0; k < MAX_CLUSTER; ++k)
            if (k < p.cluster) q += fmaf(pixels(k) * (float)p.cpg * (mk[k] - m), mk[k] - m, qk[k]);
        const float rs = 1.f / sqrtf(q / ((float)p.HW * (float)p.cpg) + p.eps);
        total[2 * g] = m;
        total[2 * g + 1] = rs;
        if (rank == 0) {
            if (p.mean) p.mean[(long long)n * p.G + g_lo + g] = m;
            if (p.rstd) p.rstd[(long long)n * p.G + g_lo + g] = rs;
        }
    }
    // also: no CTA of the cluster leaves while another reads its sums
    if (p.cluster > 1) cl.sync(); else __syncthreads();
    const ForwardOf<DT, ACT, GV> f(p, t, [&](int g) { return total[2 * (g - g_lo)]; }, [&](int g) { return total[2 * (g - g_lo) + 1]; });
    long long e = at(p, t, t.first);
    for (int s = 0; s < mine_rows; ++s, e += step) store<DT>(p.out, e, f(own<DT>(sm, s), t.nval));
}

template <int GV>
__device__ __forceinline__ void saved_normal_of(const Params& p, const Part& t, Normal<GV>& f) {
    const long long at = (long long)t.n * p.G;
    normal_of<GV>(p, t, f, [&](int g) { return p.mean[at + g]; }, [&](int g) { return p.rstd[at + g]; });
}
// minus rstd times the means of t and t xh, from pairs of means per group starting at group g0
template <int GV>
__device__ __forceinline__ void bwd_means_of(const Params& p, const Part& t, const Normal<GV>& f, const float* pairs,
                                             int g0, float (&m1)[GV], float (&m2)[GV]) {
    int g = t.c0 / p.cpg, left = p.cpg - (t.c0 - g * p.cpg);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i % (8 / GV) == 0) {
            m1[i * GV / 8] = i < t.nval ? -f.rstd[i * GV / 8] * pairs[2 * (g - g0)] : 0.f;
            m2[i * GV / 8] = i < t.nval ? -f.rstd[i * GV / 8] * pairs[2 * (g - g0) + 1] : 0.f;
        }
        if (--left == 0) { ++g; left = p.cpg; }
    }
}
// dz and xh of 8 channels of one pixel (0 for padding, whatever it holds)
template <int DT, int ACT, int GV>
__device__ __forceinline__ void bwd_terms(const Vec<DT>& vx, const Vec<DT>& vdy, const Normal<GV>& f, int nval,
                                          F2 (&dz)[4], F2 (&xh)[4]) {
    unpack<DT>(vx, xh);
    unpack<DT>(vdy, dz);
    cut(xh, nval);
    cut(dz, nval);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        xh[i] = normalised<GV>(xh[i], f, i);
        dz[i] = act_bwd<ACT>(dz[i], pre_activation<ACT, GV>(xh[i], f, i));
    }
}
// the sums that a thread keeps of them: dz, and dz xh
__device__ __forceinline__ void bwd_add(const F2 (&dz)[4], const F2 (&xh)[4], F2 (&a)[4], F2 (&b)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = add2(a[i], dz[i]);
        b[i] = fma2(dz[i], xh[i], b[i]);
    }
}
__device__ __forceinline__ void flat(const F2 (&v)[4], float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = v[i].x; f[2 * i + 1] = v[i].y; }
}
// dx = rstd (gamma dz - mean(t) - xh mean(t xh)); m1 and m2: minus the means, with their rstd
template <int DT, int GV>
__device__ __forceinline__ Vec<DT> bwd_out(const F2 (&dz)[4], const F2 (&xh)[4], const Normal<GV>& f,
                                           const float (&m1)[GV], const float (&m2)[GV]) {
    F2 d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        d[i] = fma2(mul2(dz[i], f.gamma[i]), pair_of<GV>(f.rstd, i), fma2(xh[i], pair_of<GV>(m2, i), pair_of<GV>(m1, i)));
    return pack<DT>(d);
}

// ws: per sample and channel (sum dz, sum dz xh), for gn_params_kernel
template <int DT, int ACT, int GV>
__global__ void __launch_bounds__(T, GV == 8 ? 2 : 3) gn_bwd_unit_kernel(const Params p) {
    extern __shared__ uint4 sm[];
    cg::cluster_group cl = cg::this_cluster();
    const int rank = (int)cl.block_rank(), unit = blockIdx.x / p.cluster;
    const int n = unit / p.nslab, slab = unit % p.nslab;
    const Part t = part_of(p, n, slab, rank);
    uint4* sm_dy = sm + p.iters * Elem<DT>::V16 * T;
    float* red = reinterpret_cast<float*>(sm + 2 * p.iters * Elem<DT>::V16 * T);
    float* sums = red + T * 16;             // the CTA's sums, read by the cluster
    float* total = red;                     // the unit's, once red is free
    const long long step = (long long)t.step * p.Cs;
    const int mine_rows = t.first < t.end ? (t.end - t.first + t.step - 1) / t.step : 0;
    const int half = mine_rows / 2;         // sums of the first half while the second arrives
    {
        long long e = at(p, t, t.first);
        for (int s = 0; s < mine_rows; ++s, e += step) {
            if (s == half) asm volatile("cp.async.commit_group;" ::: "memory");
            copy_in<DT>(sm, s, p.x, e);
            copy_in<DT>(sm_dy, s, p.dy, e);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    Normal<GV> f;
    saved_normal_of<GV>(p, t, f);
    F2 a2[4] = {}, b2[4] = {};
    auto take = [&](int s, int end) {
        for (; s < end; ++s) {
            F2 dz[4], xh[4];
            bwd_terms<DT, ACT, GV>(own<DT>(sm, s), own<DT>(sm_dy, s), f, t.nval, dz, xh);
            bwd_add(dz, xh, a2, b2);
        }
    };
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    take(0, half);
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    take(half, mine_rows);
    float a[8], b[8];
    flat(a2, a);
    flat(b2, b);
    reduce_columns<8>(p, a, b, red, sums);
    if (p.cluster > 1) cl.sync();
    const int c_lo = slab * p.vc * 8, nc = max(0, min(p.C - c_lo, p.vc * 8));
    for (int c = threadIdx.x; c < p.vc * 16; c += T) {
        float vk[MAX_CLUSTER], v = 0.f;     // on their way together
#pragma unroll
        for (int k = 0; k < MAX_CLUSTER; ++k) vk[k] = k < p.cluster ? cl.map_shared_rank(sums, k)[c] : 0.f;
#pragma unroll
        for (int k = 0; k < MAX_CLUSTER; ++k) v += vk[k];
        total[c] = v;
        if (rank == 0 && p.ws && c % (p.vc * 8) < nc)
            p.ws[((long long)(c / (p.vc * 8)) * p.N + n) * p.C + c_lo + c % (p.vc * 8)] = v;
    }
    if (p.cluster > 1) cl.sync(); else __syncthreads();
    float* means = total + p.vc * 16;       // the groups' mean(t) and mean(t xh)
    const float inv = 1.f / ((float)p.HW * (float)p.cpg);
    for (int g = threadIdx.x; g < nc / p.cpg; g += T) {
        float m1 = 0.f, m2 = 0.f;
        for (int c = 0; c < p.cpg; ++c) {
            const float w = p.gamma ? p.gamma[c_lo + g * p.cpg + c] : 1.f;
            m1 = fmaf(w, total[g * p.cpg + c], m1);
            m2 = fmaf(w, total[p.vc * 8 + g * p.cpg + c], m2);
        }
        means[2 * g] = m1 * inv;
        means[2 * g + 1] = m2 * inv;
    }
    __syncthreads();
    float m1[GV], m2[GV];
    bwd_means_of<GV>(p, t, f, means, c_lo / p.cpg, m1, m2);
    long long e = at(p, t, t.first);
    for (int s = 0; s < mine_rows; ++s, e += step) {
        F2 dz[4], xh[4];
        bwd_terms<DT, ACT, GV>(own<DT>(sm, s), own<DT>(sm_dy, s), f, t.nval, dz, xh);
        store<DT>(p.out, e, bwd_out<DT, GV>(dz, xh, f, m1, m2));
    }
}

// dgamma and dbeta: the samples' sums, in order
__global__ void gn_params_kernel(const float* ws, float* dgamma, float* dbeta, int N, int C) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= 2 * C) return;
    const bool second = c >= C;
    const float* s = ws + (second ? (long long)N * C : 0) + c % C;
    float v = 0.f;
#pragma unroll 8
    for (int n = 0; n < N; ++n) v += s[(long long)n * C];
    float* d = second ? dgamma : dbeta;
    if (d) d[c % C] = v;
}

// ---------------------------------------------------------------- three launches
// Grid (chunk, slab, sample). Partials at ws[sample][value][chunk][channel], value 0 and 1: mean
// and centred sum of squares (forward), sum dz and sum dz xh (backward).
__device__ __forceinline__ long long partial_at(const Params& p, int n, int value, int chunk, int c) {
    return (((long long)n * 2 + value) * p.nchunk + chunk) * p.Cs + c;
}
template <int DT, int ACT, bool BWD, int GV>
__global__ void __launch_bounds__(T, GV == 8 ? 3 : 4) gn_partial_kernel(const Params p) {
    extern __shared__ uint4 sm[];
    float* red = reinterpret_cast<float*>(sm);
    float* sums = red + T * 16;
    const Part t = part_of(p, blockIdx.z, blockIdx.y, blockIdx.x);
    if constexpr (BWD) {
        Normal<GV> f;
        saved_normal_of<GV>(p, t, f);
        F2 a2[4] = {}, b2[4] = {};
#pragma unroll 2
        for (int r = t.first; r < t.end; r += t.step) {
            F2 dz[4], xh[4];
            bwd_terms<DT, ACT, GV>(load<DT>(p.x, at(p, t, r)), load<DT>(p.dy, at(p, t, r)), f, t.nval, dz, xh);
            bwd_add(dz, xh, a2, b2);
        }
        float a[8], b[8];
        flat(a2, a);
        flat(b2, b);
        reduce_columns<8>(p, a, b, red, sums);
    } else {
        Stats<8> st;
        st.clear();
        int r = t.first;
        for (; r + 3 * t.step < t.end; r += 4 * t.step) {
            Vec<DT> q[4];
            F2 v[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = load<DT>(p.x, at(p, t, r + j * t.step));
#pragma unroll
            for (int j = 0; j < 4; ++j) unpack<DT>(q[j], v[j]);
            st.template add<4>(v);
        }
        for (; r < t.end; r += t.step) {
            F2 v[1][4];
            unpack<DT>(load<DT>(p.x, at(p, t, r)), v[0]);
            st.template add<1>(v);
        }
        block_stats<8>(p, st, (float)(min((int)(blockIdx.x + 1) * p.rows, p.HW) - (int)blockIdx.x * p.rows), red, sums);
    }
    const int c_lo = blockIdx.y * p.vc * 8;
    for (int c = threadIdx.x; c < p.vc * 8; c += T)
        if (c_lo + c < p.Cs) {
            p.ws[partial_at(p, t.n, 0, blockIdx.x, c_lo + c)] = sums[c];
            p.ws[partial_at(p, t.n, 1, blockIdx.x, c_lo + c)] = sums[p.vc * 8 + c];
        }
}

__device__ float block_sum(float v, float* sh) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < T / 32; ++w) v += sh[w];
    return v;
}
// One block per (group, sample): the chunks' and channels' statistics -> stat[sample][group]:
// forward mean and rstd, backward mean(t) and mean(t xh), with the samples' channel sums for
// gn_params_kernel in chan[value][sample][channel].
template <bool BWD>
__global__ void __launch_bounds__(T) gn_combine_kernel(const Params p, float* stat, float* chan) {
    __shared__ float sh[T / 32];
    const int g = blockIdx.x, n = blockIdx.y, c0 = g * p.cpg;
    const long long M = (long long)p.nchunk * p.cpg;
    float a = 0.f, b = 0.f;
    if constexpr (BWD) {
        // 8 lanes per channel, each a stride of the chunks, joined in lane order
        const int sub = threadIdx.x % 8;
        for (int c = threadIdx.x / 8; c - (int)threadIdx.x / 8 < p.cpg; c += T / 8) {
            float sa = 0.f, sb = 0.f;
            if (c < p.cpg)
                for (int k = sub; k < p.nchunk; k += 8) {
                    sa += p.ws[partial_at(p, n, 0, k, c0 + c)];
                    sb += p.ws[partial_at(p, n, 1, k, c0 + c)];
                }
            for (int o = 4; o; o >>= 1) {
                sa += __shfl_xor_sync(~0u, sa, o);
                sb += __shfl_xor_sync(~0u, sb, o);
            }
            if (c < p.cpg && sub == 0) {
                chan[(long long)n * p.C + c0 + c] = sa;
                chan[((long long)p.N + n) * p.C + c0 + c] = sb;
                const float w = p.gamma ? p.gamma[c0 + c] : 1.f;
                a = fmaf(w, sa, a);
                b = fmaf(w, sb, b);
            }
        }
        a = block_sum(a, sh);
        b = block_sum(b, sh);
        if (threadIdx.x == 0) {
            const float inv = 1.f / ((float)p.HW * (float)p.cpg);
            stat[2 * ((long long)n * p.G + g)] = a * inv;
            stat[2 * ((long long)n * p.G + g) + 1] = b * inv;
        }
    } else {
        for (long long i = threadIdx.x; i < M; i += T) {
            const int k = (int)(i / p.cpg), c = (int)(i % p.cpg);
            a += (float)(min((k + 1) * p.rows, p.HW) - k * p.rows) * p.ws[partial_at(p, n, 0, k, c0 + c)];
        }
        const float total = (float)p.HW * (float)p.cpg, m = block_sum(a, sh) / total;
        for (long long i = threadIdx.x; i < M; i += T) {
            const int k = (int)(i / p.cpg), c = (int)(i % p.cpg);
            const float d = p.ws[partial_at(p, n, 0, k, c0 + c)] - m;
            b += p.ws[partial_at(p, n, 1, k, c0 + c)] +
                 (float)(min((k + 1) * p.rows, p.HW) - k * p.rows) * d * d;
        }
        b = block_sum(b, sh);
        if (threadIdx.x == 0) {
            const float rs = 1.f / sqrtf(b / total + p.eps);
            const long long o = (long long)n * p.G + g;
            stat[2 * o] = m;
            stat[2 * o + 1] = rs;
            if (p.mean) p.mean[o] = m;
            if (p.rstd) p.rstd[o] = rs;
        }
    }
}
// The last chunks first: they are the ones that the partial pass left in L2.
template <int DT, int ACT, bool BWD, int GV>
__global__ void __launch_bounds__(T, GV == 8 ? 3 : 4) gn_apply_kernel(const Params p, const float* stat) {
    const Part t = part_of(p, gridDim.z - 1 - blockIdx.z, gridDim.y - 1 - blockIdx.y, gridDim.x - 1 - blockIdx.x);
    const float* s = stat + 2 * (long long)t.n * p.G;
    if constexpr (BWD) {
        Normal<GV> f;
        saved_normal_of<GV>(p, t, f);
        float m1[GV], m2[GV];
        bwd_means_of<GV>(p, t, f, s, 0, m1, m2);
#pragma unroll 2
        for (int r = t.first; r < t.end; r += t.step) {
            F2 dz[4], xh[4];
            bwd_terms<DT, ACT, GV>(load<DT>(p.x, at(p, t, r)), load<DT>(p.dy, at(p, t, r)), f, t.nval, dz, xh);
            store<DT>(p.out, at(p, t, r), bwd_out<DT, GV>(dz, xh, f, m1, m2));
        }
    } else {
        const ForwardOf<DT, ACT, GV> f(p, t, [&](int g) { return s[2 * g]; }, [&](int g) { return s[2 * g + 1]; });
#pragma unroll 4
        for (int r = t.first; r < t.end; r += t.step)
            store<DT>(p.out, at(p, t, r), f(load<DT>(p.x, at(p, t, r)), t.nval));
    }
}

// ---------------------------------------------------------------- host
static int check_shape(int nN, int nHW, int nC, int nCs, int nGroups, int nDtype) {
    if (nN < 0 || nHW <= 0 || nC <= 0 || nCs < nC || nCs % 8 || nGroups <= 0 || nC % nGroups)
        return OM_ERR_INVALID;
    if (nDtype != OM_DTYPE_F32 && nDtype != OM_DTYPE_BF16 && nDtype != OM_DTYPE_F16)
        return OM_ERR_UNSUPPORTED;
    if (nHW > (1 << 30)) return OM_ERR_UNSUPPORTED;
    return OM_OK;
}
static bool aligned(const void* p, int a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// GV of a number of channels per group. Other multiples of 4 than these could keep two entries as well;
// only 4 and multiples of 8, the usual ones, were measured so, and the rest take the general form
static int entries(int cpg) { return cpg % 8 == 0 ? 1 : cpg == 4 ? 2 : 8; }

// Fills in the split of the work: p->cluster > 0 for the one-launch form with `smem` bytes,
// 0 for the three-launch form.
static void plan(Params* p, int dtype, bool bwd, size_t* smem) {
    const int size = dtype == OM_DTYPE_F32 ? 4 : 2;
    p->cpg = p->C / p->G;
    // whole groups in whole vectors, 64 bytes of a pixel where the channels give as many
    long long unit = p->cpg;
    int gcd = 8;
    while (unit % gcd) gcd /= 2;
    unit *= 8 / gcd;
    long long slab = unit;
    while (slab * size < 64 && slab < p->C) slab += unit;
    if (slab >= p->C) slab = p->Cs;
    const int per_vec = 8 * size * (bwd ? 2 : 1);        // bytes kept for a vector
    p->cluster = 0;
    if (slab / 8 <= MAX_VC) {
        p->vc = (int)(slab / 8);
        p->nslab = (int)((p->Cs + slab - 1) / slab);
        const int step = T / p->vc;
        const int nv = bwd ? 8 : entries(p->cpg);
        const size_t fixed = (size_t)(T + p->vc) * 2 * nv * 4 + (bwd ? 0 : 4 * MAX_GROUPS * 4);
        for (int k = 1; k <= MAX_CLUSTER; k *= 2) {
            const int rows = (p->HW + k - 1) / k, iters = (rows + step - 1) / step;
            const size_t need = (size_t)iters * T * per_vec + fixed;
            // one CTA on an SM leaves loads, sums and stores one after another: only for one wave
            if (need > ((long long)p->N * p->nslab * k <= 148 ? SMEM_MAX : KEEP_MAX)) continue;
            p->cluster = k; p->rows = rows; p->iters = iters; *smem = need;
            // enough parts to fill the GPU, with two CTAs on an SM
            if ((long long)p->N * p->nslab * k >= 2 * 148 && need <= KEEP_GOOD) break;
            if (iters <= 4) break;
        }
    }
    if (p->cluster) return;
    p->vc = p->Cs / 8 < MAX_VC ? p->Cs / 8 : MAX_VC;
    p->nslab = (p->Cs / 8 + p->vc - 1) / p->vc;
    const int step = T / p->vc;
    int iters = 8;
    while (iters < 256 && (long long)p->N * p->nslab * ((p->HW + step * iters - 1) / (step * iters)) > 148 * 16) iters *= 2;
    p->rows = step * iters;
    p->iters = iters;
    p->nchunk = (p->HW + p->rows - 1) / p->rows;
    *smem = (size_t)T * 16 * 4 + (size_t)p->vc * 16 * 4;
}
static long long ws_floats(const Params& p, bool bwd) {
    const long long chan = bwd ? 2LL * p.N * p.C : 0;
    if (p.cluster) return chan;
    return chan + 2LL * p.N * p.G + 2LL * p.N * p.nchunk * p.Cs;
}

template <int DT, int ACT, bool BWD>
static int launch(DeviceCtx* c, Params p, size_t smem) {
    static bool attr_set[64] = {false};
    if (p.cluster) {
        using Kern = void (*)(const Params);
        const Kern kerns[3] = {BWD ? gn_bwd_unit_kernel<DT, ACT, 1> : gn_fwd_unit_kernel<DT, ACT, 1>,
                               BWD ? gn_bwd_unit_kernel<DT, ACT, 2> : gn_fwd_unit_kernel<DT, ACT, 2>,
                               BWD ? gn_bwd_unit_kernel<DT, ACT, 8> : gn_fwd_unit_kernel<DT, ACT, 8>};
        if (!attr_set[c->device]) {
            for (Kern k : kerns)
                OMB_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX));
            attr_set[c->device] = true;
        }
        const int gv = entries(p.cpg);
        const Kern kern = kerns[gv == 1 ? 0 : gv == 2 ? 1 : 2];
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((long long)p.N * p.nslab * p.cluster));
        cfg.blockDim = dim3(T);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = c->compute;
        cudaLaunchAttribute a[1];
        a[0].id = cudaLaunchAttributeClusterDimension;
        a[0].val.clusterDim.x = p.cluster;
        a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
        cfg.attrs = a;
        cfg.numAttrs = 1;
        OMB_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
        if (after_launch(c) != OM_OK) return OM_ERR_CUDA;
    } else {
        float* chan = p.ws;
        float* stat = chan + (BWD ? 2LL * p.N * p.C : 0);
        p.ws = stat + 2LL * p.N * p.G;
        const dim3 grid(p.nchunk, p.nslab, p.N);
        const int gv = BWD ? entries(p.cpg) : 8;
        (gv == 1   ? gn_partial_kernel<DT, ACT, BWD, BWD ? 1 : 8>
         : gv == 2 ? gn_partial_kernel<DT, ACT, BWD, BWD ? 2 : 8>
                   : gn_partial_kernel<DT, ACT, BWD, 8>)<<<grid, T, smem, c->compute>>>(p);
        if (after_launch(c) != OM_OK) return OM_ERR_CUDA;
        gn_combine_kernel<BWD><<<dim3(p.G, p.N), T, 0, c->compute>>>(p, stat, chan);
        if (after_launch(c) != OM_OK) return OM_ERR_CUDA;
        (gv == 1   ? gn_apply_kernel<DT, ACT, BWD, BWD ? 1 : 8>
         : gv == 2 ? gn_apply_kernel<DT, ACT, BWD, BWD ? 2 : 8>
                   : gn_apply_kernel<DT, ACT, BWD, 8>)<<<grid, T, 0, c->compute>>>(p, stat);
        if (after_launch(c) != OM_OK) return OM_ERR_CUDA;
        p.ws = chan;
    }
    if (BWD && (p.dgamma || p.dbeta)) {
        gn_params_kernel<<<(2 * p.C + 127) / 128, 128, 0, c->compute>>>(p.ws, p.dgamma, p.dbeta, p.N, p.C);
        return after_launch(c);
    }
    return OM_OK;
}
template <int DT, bool BWD>
static int launch_act(DeviceCtx* c, const Params& p, size_t smem, int act) {
    switch (act) {
        case OM_ACT_NONE: return launch<DT, OM_ACT_NONE, BWD>(c, p, smem);
        case OM_ACT_RELU: return launch<DT, OM_ACT_RELU, BWD>(c, p, smem);
        case OM_ACT_RELU6: return launch<DT, OM_ACT_RELU6, BWD>(c, p, smem);
        default: return launch<DT, OM_ACT_SILU, BWD>(c, p, smem);
    }
}
template <bool BWD>
static int dispatch(DeviceCtx* c, Params p, int act, int dtype) {
    size_t smem = 0;
    plan(&p, dtype, BWD, &smem);
    if (ws_floats(p, BWD) > 0 && (!p.ws || !aligned(p.ws, 16))) return OM_ERR_INVALID;
    if (p.cluster ? (long long)p.N * p.nslab * p.cluster > 0x7FFFFFFF : p.N > 65535)
        return OM_ERR_UNSUPPORTED;      // the grid's limits
    if (dtype == OM_DTYPE_F32) return launch_act<OM_DTYPE_F32, BWD>(c, p, smem, act);
    if (dtype == OM_DTYPE_BF16) return launch_act<OM_DTYPE_BF16, BWD>(c, p, smem, act);
    return launch_act<OM_DTYPE_F16, BWD>(c, p, smem, act);
}

}  // namespace gn
}  // namespace omb

using namespace omb;

extern "C" long long omCudaGroupNormNhwcWorkspaceBytes(int nN, int nHW, int nC, int nCs,
                                                       int nGroups, int nDtype, int bBackward) {
    const int st = gn::check_shape(nN, nHW, nC, nCs, nGroups, nDtype);
    if (st != OM_OK) return st;
    gn::Params p = {};
    p.N = nN; p.HW = nHW; p.C = nC; p.Cs = nCs; p.G = nGroups;
    size_t smem;
    gn::plan(&p, nDtype, bBackward != 0, &smem);
    return gn::ws_floats(p, bBackward != 0) * 4;
}

extern "C" int omCudaGroupNormActNhwc(const void* pIn, void* pOut, const float* pGamma,
                                      const float* pBeta, float* pMean, float* pInvStd,
                                      void* pWorkspace, int nN, int nHW, int nC, int nCs,
                                      int nGroups, float fEps, int nAct, int nDtype) {
    OMB_CTX_OR_FAIL(c);
    const int st = gn::check_shape(nN, nHW, nC, nCs, nGroups, nDtype);
    if (st != OM_OK) return st;
    if (!(fEps >= 0.f) || nAct < OM_ACT_NONE || nAct > OM_ACT_SILU) return OM_ERR_INVALID;
    if (nN == 0) return OM_OK;
    if (!pIn || !pOut || !gn::aligned(pIn, 16) || !gn::aligned(pOut, 16)) return OM_ERR_INVALID;
    gn::Params p = {};
    p.x = pIn; p.out = pOut; p.gamma = pGamma; p.beta = pBeta; p.mean = pMean; p.rstd = pInvStd;
    p.ws = static_cast<float*>(pWorkspace);
    p.N = nN; p.HW = nHW; p.C = nC; p.Cs = nCs; p.G = nGroups; p.eps = fEps;
    return gn::dispatch<false>(c, p, nAct, nDtype);
}

extern "C" int omCudaGroupNormActNhwcBackward(const void* pGradOut, const void* pIn,
                                              const float* pMean, const float* pInvStd,
                                              const float* pGamma, const float* pBeta,
                                              void* pGradIn, float* pGradGamma, float* pGradBeta,
                                              void* pWorkspace, int nN, int nHW, int nC, int nCs,
                                              int nGroups, int nAct, int nDtype) {
    OMB_CTX_OR_FAIL(c);
    const int st = gn::check_shape(nN, nHW, nC, nCs, nGroups, nDtype);
    if (st != OM_OK) return st;
    if (nAct < OM_ACT_NONE || nAct > OM_ACT_SILU) return OM_ERR_INVALID;
    if (nN == 0) {
        if (pGradGamma) OMB_CHECK(cudaMemsetAsync(pGradGamma, 0, sizeof(float) * nC, c->compute));
        if (pGradBeta) OMB_CHECK(cudaMemsetAsync(pGradBeta, 0, sizeof(float) * nC, c->compute));
        return OM_OK;
    }
    if (!pGradOut || !pIn || !pMean || !pInvStd || !pGradIn || !gn::aligned(pGradOut, 16) ||
        !gn::aligned(pIn, 16) || !gn::aligned(pGradIn, 16))
        return OM_ERR_INVALID;
    gn::Params p = {};
    p.x = pIn; p.dy = pGradOut; p.out = pGradIn; p.gamma = pGamma; p.beta = pBeta;
    p.mean = const_cast<float*>(pMean); p.rstd = const_cast<float*>(pInvStd);
    p.dgamma = pGradGamma; p.dbeta = pGradBeta;
    p.ws = static_cast<float*>(pWorkspace);
    p.N = nN; p.HW = nHW; p.C = nC; p.Cs = nCs; p.G = nGroups;
    return gn::dispatch<true>(c, p, nAct, nDtype);
}
