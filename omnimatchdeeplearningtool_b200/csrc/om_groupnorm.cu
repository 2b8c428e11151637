// GroupNorm with its activation on channels-last maps, forward and backward.
#include "om_common.cuh"

namespace omb {
namespace gn {

template <int DT> struct Elem { using T = float; };
template <> struct Elem<OM_DTYPE_BF16> { using T = __nv_bfloat16; };
template <> struct Elem<OM_DTYPE_F16> { using T = __half; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(float v, __half& o) { o = __float2half_rn(v); }

__device__ __forceinline__ float act_fwd(float z, int act) {
    if (act == OM_ACT_SILU) return z / (1.f + __expf(-z));
    return apply_act(z, act);
}
// dz = dy * act'(z)
__device__ __forceinline__ float act_bwd(float dy, float z, int act) {
    if (act == OM_ACT_SILU) {
        const float s = 1.f / (1.f + __expf(-z));
        return dy * (s * (1.f + z * (1.f - s)));
    }
    if (act == OM_ACT_RELU) return z > 0.f ? dy : 0.f;
    if (act == OM_ACT_RELU6) return z > 0.f && z < 6.f ? dy : 0.f;
    return dy;
}

struct Params {
    const void* x;
    const void* dy;
    void* out;
    const float *gamma, *beta;
    float *mean, *rstd;   // forward: written when given
    float *dgamma, *dbeta;
    int N, HW, C, Cs, G, act;
    float eps;
};

// Sum over the block (blockDim.x a multiple of 32), the result in every thread.
__device__ float block_sum(float v, float* sh) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < (int)blockDim.x / 32; ++w) v += sh[w];
    return v;
}

// One block per (sample, group); group G stands for the stored channels past C, which become 0.
template <int DT>
__global__ void gn_fwd_kernel(const Params p) {
    using T = typename Elem<DT>::T;
    __shared__ float sh[32];
    const int n = blockIdx.x / (p.G + 1), g = blockIdx.x % (p.G + 1);
    const T* x = static_cast<const T*>(p.x) + (long long)n * p.HW * p.Cs;
    T* y = static_cast<T*>(p.out) + (long long)n * p.HW * p.Cs;
    if (g == p.G) {
        const int pad = p.Cs - p.C;
        for (long long i = threadIdx.x; i < (long long)p.HW * pad; i += blockDim.x)
            y[i / pad * p.Cs + p.C + i % pad] = T(0.f);
        return;
    }
    const int cpg = p.C / p.G, c0 = g * cpg;
    const long long M = (long long)p.HW * cpg;
    float s = 0.f;
    for (long long i = threadIdx.x; i < M; i += blockDim.x)
        s += to_f(x[i / cpg * p.Cs + c0 + i % cpg]);
    const float mean = block_sum(s, sh) / (float)M;
    s = 0.f;
    for (long long i = threadIdx.x; i < M; i += blockDim.x) {
        const float d = to_f(x[i / cpg * p.Cs + c0 + i % cpg]) - mean;
        s += d * d;
    }
    const float rstd = rsqrtf(block_sum(s, sh) / (float)M + p.eps);
    if (threadIdx.x == 0) {
        if (p.mean) p.mean[n * p.G + g] = mean;
        if (p.rstd) p.rstd[n * p.G + g] = rstd;
    }
    for (long long i = threadIdx.x; i < M; i += blockDim.x) {
        const int c = c0 + (int)(i % cpg);
        const long long at = i / cpg * p.Cs + c;
        const float xh = (to_f(x[at]) - mean) * rstd;
        from_f(act_fwd(xh * (p.gamma ? p.gamma[c] : 1.f) + (p.beta ? p.beta[c] : 0.f), p.act), y[at]);
    }
}

template <int DT>
__device__ __forceinline__ void bwd_point(const Params& p, long long at, int c, float mean,
                                          float rstd, float& dz, float& xh) {
    using T = typename Elem<DT>::T;
    xh = (to_f(static_cast<const T*>(p.x)[at]) - mean) * rstd;
    const float z = xh * (p.gamma ? p.gamma[c] : 1.f) + (p.beta ? p.beta[c] : 0.f);
    dz = act_bwd(to_f(static_cast<const T*>(p.dy)[at]), z, p.act);
}

// Per channel: dgamma and dbeta over samples and pixels.
template <int DT>
__global__ void gn_bwd_params_kernel(const Params p) {
    __shared__ float sh[32];
    const int c = blockIdx.x, g = c / (p.C / p.G);
    float a = 0.f, b = 0.f;
    for (long long i = threadIdx.x; i < (long long)p.N * p.HW; i += blockDim.x) {
        const int n = (int)(i / p.HW);
        float dz, xh;
        bwd_point<DT>(p, i * p.Cs + c, c, p.mean[n * p.G + g], p.rstd[n * p.G + g], dz, xh);
        a += dz * xh;
        b += dz;
    }
    a = block_sum(a, sh);
    b = block_sum(b, sh);
    if (threadIdx.x == 0) {
        if (p.dgamma) p.dgamma[c] = a;
        if (p.dbeta) p.dbeta[c] = b;
    }
}

template <int DT>
__global__ void gn_bwd_kernel(const Params p) {
    using T = typename Elem<DT>::T;
    __shared__ float sh[32];
    const int n = blockIdx.x / (p.G + 1), g = blockIdx.x % (p.G + 1);
    const long long base = (long long)n * p.HW * p.Cs;
    T* dx = static_cast<T*>(p.out);
    if (g == p.G) {
        const int pad = p.Cs - p.C;
        for (long long i = threadIdx.x; i < (long long)p.HW * pad; i += blockDim.x)
            dx[base + i / pad * p.Cs + p.C + i % pad] = T(0.f);
        return;
    }
    const int cpg = p.C / p.G, c0 = g * cpg;
    const long long M = (long long)p.HW * cpg;
    const float mean = p.mean[n * p.G + g], rstd = p.rstd[n * p.G + g];
    float a = 0.f, b = 0.f;
    for (long long i = threadIdx.x; i < M; i += blockDim.x) {
        const int c = c0 + (int)(i % cpg);
        float dz, xh;
        bwd_point<DT>(p, base + i / cpg * p.Cs + c, c, mean, rstd, dz, xh);
        const float t = dz * (p.gamma ? p.gamma[c] : 1.f);
        a += t;
        b += t * xh;
    }
    a = block_sum(a, sh) / (float)M;
    b = block_sum(b, sh) / (float)M;
    for (long long i = threadIdx.x; i < M; i += blockDim.x) {
        const int c = c0 + (int)(i % cpg);
        const long long at = base + i / cpg * p.Cs + c;
        float dz, xh;
        bwd_point<DT>(p, at, c, mean, rstd, dz, xh);
        from_f(rstd * (dz * (p.gamma ? p.gamma[c] : 1.f) - a - xh * b), dx[at]);
    }
}

static int check_shape(int nN, int nHW, int nC, int nCs, int nGroups, int nDtype) {
    if (nN < 0 || nHW <= 0 || nC <= 0 || nCs < nC || nCs % 8 || nGroups <= 0 || nC % nGroups)
        return OM_ERR_INVALID;
    if (nDtype != OM_DTYPE_F32 && nDtype != OM_DTYPE_BF16 && nDtype != OM_DTYPE_F16)
        return OM_ERR_UNSUPPORTED;
    return OM_OK;
}
static bool aligned(const void* p, int a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

}  // namespace gn
}  // namespace omb

using namespace omb;

extern "C" long long omCudaGroupNormNhwcWorkspaceBytes(int nN, int nHW, int nC, int nCs,
                                                       int nGroups, int nDtype, int bBackward) {
    const int st = gn::check_shape(nN, nHW, nC, nCs, nGroups, nDtype);
    return st != OM_OK ? st : 0;
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
    p.N = nN; p.HW = nHW; p.C = nC; p.Cs = nCs; p.G = nGroups; p.act = nAct; p.eps = fEps;
    const int grid = nN * (nGroups + 1);
    if (nDtype == OM_DTYPE_F32)
        gn::gn_fwd_kernel<OM_DTYPE_F32><<<grid, 256, 0, c->compute>>>(p);
    else if (nDtype == OM_DTYPE_BF16)
        gn::gn_fwd_kernel<OM_DTYPE_BF16><<<grid, 256, 0, c->compute>>>(p);
    else
        gn::gn_fwd_kernel<OM_DTYPE_F16><<<grid, 256, 0, c->compute>>>(p);
    return after_launch(c);
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
    p.N = nN; p.HW = nHW; p.C = nC; p.Cs = nCs; p.G = nGroups; p.act = nAct;
    const int grid = nN * (nGroups + 1);
    if (pGradGamma || pGradBeta) {  // before dX, which may overwrite dY
        if (nDtype == OM_DTYPE_F32)
            gn::gn_bwd_params_kernel<OM_DTYPE_F32><<<nC, 256, 0, c->compute>>>(p);
        else if (nDtype == OM_DTYPE_BF16)
            gn::gn_bwd_params_kernel<OM_DTYPE_BF16><<<nC, 256, 0, c->compute>>>(p);
        else
            gn::gn_bwd_params_kernel<OM_DTYPE_F16><<<nC, 256, 0, c->compute>>>(p);
        if (after_launch(c) != OM_OK) return OM_ERR_CUDA;
    }
    if (nDtype == OM_DTYPE_F32)
        gn::gn_bwd_kernel<OM_DTYPE_F32><<<grid, 256, 0, c->compute>>>(p);
    else if (nDtype == OM_DTYPE_BF16)
        gn::gn_bwd_kernel<OM_DTYPE_BF16><<<grid, 256, 0, c->compute>>>(p);
    else
        gn::gn_bwd_kernel<OM_DTYPE_F16><<<grid, 256, 0, c->compute>>>(p);
    return after_launch(c);
}
