// topk_device.h -- what the top-logit kernels (topk_select.hip, topk_kl.hip) share: groups of threads that own a row, and the running
// (maximum, sum) of a softmax whose terms may be -inf.
#pragma once
#include <float.h>

#include "cgd_device.h"

namespace sd {

constexpr int kTopkMax = 128;            // most entries per row
constexpr int kTopkMaxClasses = 262144;  // membership bits of a row stay within 32 KB of LDS
constexpr long kMaxBlocks = 0xffffff;    // of 256 threads: a launch holds fewer than 2^32 threads
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kTauMin = 1e-38f, kTauMax = 1e38f;      // log2(e) / tau is a normal number

// A row belongs to NT threads: one wave (four rows per workgroup) or a whole workgroup.  Waves of a workgroup work on rows of their own when
// NT == 64, so that form must not use the workgroup barrier: LDS operations of one wave execute in order, only the compiler is held back.
template <int NT>
__device__ __forceinline__ void group_sync() {
    if constexpr (NT == 64) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    } else {
        __syncthreads();
    }
}

// (m, s): s = sum of 2^{(x - m) c2} over the terms seen, m their maximum; nothing seen (or only -inf): (-inf, 0).
struct Online {
    float m, s;
};
// -inf - (-inf) is never formed.  A maximum of +inf makes s NaN, as it does a softmax; with SUM the sum itself is wanted, and it is inf.
template <bool SUM = false>
__device__ __forceinline__ float finite_ref(float m) {
    return m == -INFINITY ? 0.f : (SUM ? fminf(m, FLT_MAX) : m);
}
template <bool SUM = false, int N>
__device__ __forceinline__ void online_fold(Online &o, const float (&x)[N], float c2) {
    float m = o.m;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[i]);
    const float r = finite_ref<SUM>(m);
    float s = o.s * ex2((o.m - r) * c2);
#pragma unroll
    for (int i = 0; i < N; ++i) s += ex2((x[i] - r) * c2);
    o.m = m;
    o.s = s;
}
template <bool SUM = false>
__device__ __forceinline__ Online online_merge(Online a, Online b, float c2) {
    const float m = fmaxf(a.m, b.m), r = finite_ref<SUM>(m);
    return {m, a.s * ex2((a.m - r) * c2) + b.s * ex2((b.m - r) * c2)};
}
// over the NT threads of a group, the same value in all of them; `tmp` holds NT / 64 entries.  A butterfly: the order of the sum is fixed.
template <int NT, bool SUM = false>
__device__ __forceinline__ Online online_group(Online o, Online *tmp, int tid, float c2) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const Online p = {__shfl_xor(o.m, d, 64), __shfl_xor(o.s, d, 64)};
        o = online_merge<SUM>(o, p, c2);
    }
    if constexpr (NT > 64) {
        if ((tid & 63) == 0) tmp[tid >> 6] = o;
        __syncthreads();
        o = tmp[0];
#pragma unroll
        for (int w = 1; w < NT / 64; ++w) o = online_merge<SUM>(o, tmp[w], c2);
        __syncthreads();
    }
    return o;
}

template <typename T>
__device__ __forceinline__ void unpack_vec(typename VecIO<T>::raw_t r, float (&a)[VecIO<T>::N]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if constexpr (sizeof(T) == 4) a[q] = r[q];
        else a[2 * q] = __uint_as_float((unsigned)r[q] << 16), a[2 * q + 1] = __uint_as_float((unsigned)r[q] & 0xffff0000u);
    }
}

// Elements that come before the first 16-byte boundary of a row.
template <typename T>
__device__ __forceinline__ int row_head(const T *row, int n) {
    const int off = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    return off < n ? off : n;
}

}  // namespace sd
