// Attention and its backward, which recomputes the probabilities from the saved log-sum-exp.
#include "om_common.cuh"

namespace omb {
namespace attn {

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

// One block per (batch, head, query): 128 keys at a time, thread t their scores, then column t
// of the output.
template <int DT>
__global__ void __launch_bounds__(128) attn_fwd_kernel(const Params p) {
    using H16 = Half16<DT>;
    __shared__ float sp[128], sh[4];
    const int i = blockIdx.x, h = blockIdx.y % p.H, b = blockIdx.y / p.H, t = threadIdx.x;
    const int hk = h / (p.H / p.Hkv);
    const int ql = len_of(p.qlens, b, p.Sq), kl = len_of(p.kvlens, b, p.Sk);
    int end = i < ql ? kl : 0;
    if (p.causal) end = min(end, i + kl - ql + 1);
    const auto* q = row<DT>(p.q, b, i, h);
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int j0 = 0; j0 < end; j0 += 128) {
        const int j = j0 + t;
        const float s = j < end ? dot<DT>(q, row<DT>(p.k, b, j, hk), p.D) * p.scale : -INFINITY;
        const float m2 = fmaxf(m, block_reduce(s, sh, true));
        const float w = j < end ? expf(s - m2) : 0.f, corr = expf(m - m2);
        l = l * corr + block_reduce(w, sh, false);
        m = m2;
        sp[t] = w;
        __syncthreads();
        if (t < p.D) {
            acc *= corr;
            for (int jj = 0; jj < min(128, end - j0); ++jj)
                acc += sp[jj] * H16::to_f(row<DT>(p.v, b, j0 + jj, hk)[t]);
        }
    }
    if (t < p.D) row_out<DT>(p.o, b, i, h)[t] = H16::from_f(l > 0.f ? acc / l : 0.f);
    if (t == 0 && p.lse)
        p.lse[((long long)b * p.H + h) * p.Sq + i] = l > 0.f ? m + logf(l) : -INFINITY;
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
    attn::Params p = {};
    if (!pStrides || !attn::view(&p.q, pQ, pStrides, nBatch, nSq, nHeads) ||
        !attn::view(&p.k, pK, pStrides + 3, nBatch, nSk, nKvHeads) ||
        !attn::view(&p.v, pV, pStrides + 6, nBatch, nSk, nKvHeads) ||
        !attn::view(&p.o, pOut, pStrides + 9, nBatch, nSq, nHeads))
        return OM_ERR_INVALID;
    if (nBatch == 0 || nSq == 0) return OM_OK;
    p.lse = pLse; p.qlens = pQLens; p.kvlens = pKvLens;
    p.B = nBatch; p.H = nHeads; p.Hkv = nKvHeads; p.Sq = nSq; p.Sk = nSk; p.D = nHeadDim;
    p.causal = bCausal != 0; p.scale = fScale;
    const dim3 grid(nSq, nBatch * nHeads);
    if (nDtype == OM_DTYPE_BF16)
        attn::attn_fwd_kernel<OM_DTYPE_BF16><<<grid, 128, 0, c->compute>>>(p);
    else
        attn::attn_fwd_kernel<OM_DTYPE_F16><<<grid, 128, 0, c->compute>>>(p);
    return after_launch(c);
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
    p.causal = bCausal != 0; p.scale = fScale;
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
