// Dropout with the residual add from a counter-based generator (omCudaDropoutAdd): the mask is
// a function of (seed, offset, element index), so it is never stored and the backward pass
// draws it again. A captured call keeps the arguments it was captured with, so
// omCudaDropoutAddStep adds to the offset a step that the kernel reads.
//
// Element i takes 16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011) at counter (i / 8, offset): one generator call serves
// the 8 elements of a 16-byte vector. 16 bits give the drop probability in steps of 2^-16; the
// scale is 65536 / (65536 - T) for the T that is used, so the expectation stays exact.
#include "om_common.cuh"

namespace omb {
namespace drop {

__device__ __forceinline__ uint4 philox4x32_10(uint4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long p0 = (unsigned long long)c.x * 0xD2511F53u;
        const unsigned long long p1 = (unsigned long long)c.z * 0xCD9E8D57u;
        c = make_uint4((uint32_t)(p1 >> 32) ^ c.y ^ k0, (uint32_t)p1,
                       (uint32_t)(p0 >> 32) ^ c.w ^ k1, (uint32_t)p0);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return c;
}

template <int DT> struct Elem { using T = float; };
template <> struct Elem<OM_DTYPE_BF16> { using T = __nv_bfloat16; };
template <> struct Elem<OM_DTYPE_F16> { using T = __half; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(float v, __half& o) { o = __float2half_rn(v); }

struct Params {
    const void* x;
    const void* res;
    void* out;
    long long n;
    uint32_t k0, k1, o0, o1;
    uint32_t thr;   // T: elements whose 16 bits are below it are dropped
    float scale;
    const unsigned long long* step;   // STEP: added to the offset
};

template <class T> struct alignas(16) Eight { T v[8]; };

// The 8 elements of group g: kept and scaled, or dropped, plus the residual
template <class T, bool RES>
__device__ __forceinline__ void dropout_group(const Params& p, uint32_t o0, uint32_t o1, long long g, Eight<T>& x, const Eight<T>& r) {
    const uint4 w = philox4x32_10(make_uint4((uint32_t)g, (uint32_t)(g >> 32), o0, o1), p.k0, p.k1);
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t bits = j % 2 ? word[j / 2] >> 16 : word[j / 2] & 0xFFFFu;
        float y = bits >= p.thr ? to_f(x.v[j]) * p.scale : 0.f;
        if (RES) y += to_f(r.v[j]);
        from_f(y, x.v[j]);
    }
}

// One thread per 8 elements, four groups in flight (fp32: two): the loads of all go out before the first
// group's generator rounds (with one, 56 us for 50 M f16 elements whose copy takes 31 us; the
// rounds alone are about half of that in issue slots). VEC: all pointers 16-byte aligned, so full
// groups move in 16-byte accesses; the last group, and every group otherwise, goes element by
// element. STEP: a variant of its own, so that the others' offset stays two constants (as a 64-bit
// register 42.5 -> 43.8 us for those elements).
template <int DT, bool RES, bool VEC, bool STEP>
__global__ void __launch_bounds__(256) dropout_kernel(const Params p) {
    using T = typename Elem<DT>::T;
    constexpr int U = DT == OM_DTYPE_F32 ? 2 : 4;
    const T* x = static_cast<const T*>(p.x);
    const T* res = static_cast<const T*>(p.res);
    T* out = static_cast<T*>(p.out);
    const long long groups = (p.n + 7) / 8, whole = p.n / 8, stride = gridDim.x * 256LL;
    uint32_t o0 = p.o0, o1 = p.o1;
    if (STEP) {
        const unsigned long long offset = ((unsigned long long)o1 << 32 | o0) + *p.step;
        o0 = (uint32_t)offset;
        o1 = (uint32_t)(offset >> 32);
    }
    long long g = blockIdx.x * 256LL + threadIdx.x;
    if (VEC) {
        for (; g + (U - 1) * stride < whole; g += U * stride) {
            Eight<T> v[U], r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
                    reinterpret_cast<uint4*>(&v[u])[j] = reinterpret_cast<const uint4*>(x + (g + u * stride) * 8)[j];
                    if (RES) reinterpret_cast<uint4*>(&r[u])[j] = reinterpret_cast<const uint4*>(res + (g + u * stride) * 8)[j];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                dropout_group<T, RES>(p, o0, o1, g + u * stride, v[u], r[u]);
#pragma unroll
                for (int j = 0; j < (int)sizeof(T) / 2; ++j)
                    reinterpret_cast<uint4*>(out + (g + u * stride) * 8)[j] = reinterpret_cast<uint4*>(&v[u])[j];
            }
        }
    }
    for (; g < groups; g += stride) {
        Eight<T> v, r;
        const long long i0 = g * 8;
        const int left = p.n - i0 < 8 ? (int)(p.n - i0) : 8;
        if (VEC && left == 8) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
                reinterpret_cast<uint4*>(&v)[j] = reinterpret_cast<const uint4*>(x + i0)[j];
                if (RES) reinterpret_cast<uint4*>(&r)[j] = reinterpret_cast<const uint4*>(res + i0)[j];
            }
        } else {
            for (int j = 0; j < 8; ++j) {
                v.v[j] = j < left ? x[i0 + j] : T(0.f);
                if (RES) r.v[j] = j < left ? res[i0 + j] : T(0.f);
            }
        }
        dropout_group<T, RES>(p, o0, o1, g, v, r);
        if (VEC && left == 8) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; ++j)
                reinterpret_cast<uint4*>(out + i0)[j] = reinterpret_cast<uint4*>(&v)[j];
        } else {
            for (int j = 0; j < left; ++j) out[i0 + j] = v.v[j];
        }
    }
}

template <int DT, bool RES>
static void launch(DeviceCtx* c, const Params& p, bool vec) {
    // 16-bit: 8 CTAs an SM that go round; fp32: 8192 elements a CTA (50 M elements: 42 and 44 us the
    // two ways in 16 bits, 75 and 66 us in fp32)
    const long long ctas = (p.n + 8191) / 8192;
    const int grid = DT == OM_DTYPE_F32 && ctas <= 0x7FFFFFFF ? (int)ctas : ew_grid(c, (p.n + 7) / 8, 256);
    auto kern = p.step ? (vec ? dropout_kernel<DT, RES, true, true> : dropout_kernel<DT, RES, false, true>)
                       : (vec ? dropout_kernel<DT, RES, true, false> : dropout_kernel<DT, RES, false, false>);
    kern<<<grid, 256, 0, c->compute>>>(p);
}

static int dropout_add(const void* pIn, const void* pResidual, void* pOut, long long nCount, float fProb,
                       unsigned long long nSeed, unsigned long long nOffset, const unsigned long long* pStep,
                       int nDtype) {
    OMB_CTX_OR_FAIL(c);
    if (nCount < 0 || !(fProb >= 0.f && fProb <= 1.f)) return OM_ERR_INVALID;
    if (nDtype != OM_DTYPE_F32 && nDtype != OM_DTYPE_BF16 && nDtype != OM_DTYPE_F16)
        return OM_ERR_UNSUPPORTED;
    if (nCount == 0) return OM_OK;
    const uintptr_t any = reinterpret_cast<uintptr_t>(pIn) | reinterpret_cast<uintptr_t>(pOut) |
                          reinterpret_cast<uintptr_t>(pResidual);
    if (!pIn || !pOut || any % (nDtype == OM_DTYPE_F32 ? 4 : 2)) return OM_ERR_INVALID;
    Params p;
    p.x = pIn; p.res = pResidual; p.out = pOut; p.n = nCount;
    p.k0 = (uint32_t)nSeed; p.k1 = (uint32_t)(nSeed >> 32);
    p.o0 = (uint32_t)nOffset; p.o1 = (uint32_t)(nOffset >> 32);
    p.step = pStep;
    p.thr = (uint32_t)((double)fProb * 65536.0 + 0.5);
    p.scale = p.thr < 65536 ? (float)(65536.0 / (65536.0 - p.thr)) : 0.f;
    const bool vec = any % 16 == 0;
    const bool res = pResidual != nullptr;
    if (nDtype == OM_DTYPE_F32)
        res ? launch<OM_DTYPE_F32, true>(c, p, vec) : launch<OM_DTYPE_F32, false>(c, p, vec);
    else if (nDtype == OM_DTYPE_BF16)
        res ? launch<OM_DTYPE_BF16, true>(c, p, vec) : launch<OM_DTYPE_BF16, false>(c, p, vec);
    else
        res ? launch<OM_DTYPE_F16, true>(c, p, vec) : launch<OM_DTYPE_F16, false>(c, p, vec);
    return after_launch(c);
}

}  // namespace drop
}  // namespace omb

extern "C" int omCudaDropoutAdd(const void* pIn, const void* pResidual, void* pOut,
                                long long nCount, float fProb, unsigned long long nSeed,
                                unsigned long long nOffset, int nDtype) {
    return omb::drop::dropout_add(pIn, pResidual, pOut, nCount, fProb, nSeed, nOffset, nullptr, nDtype);
}

extern "C" int omCudaDropoutAddStep(const void* pIn, const void* pResidual, void* pOut,
                                    long long nCount, float fProb, unsigned long long nSeed,
                                    unsigned long long nOffset, const unsigned long long* pStep,
                                    int nDtype) {
    OMB_CTX_OR_FAIL(c);
    if (!pStep || reinterpret_cast<uintptr_t>(pStep) % 8) return OM_ERR_INVALID;
    return omb::drop::dropout_add(pIn, pResidual, pOut, nCount, fProb, nSeed, nOffset, pStep, nDtype);
}
