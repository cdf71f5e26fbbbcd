// window_train.hip -- window multi-head self-attention with a learned bias, forward and backward (a Swin student's blocks), gfx950.
//
// Reference: mmseg/models/backbones/swin_transformer.py:119-153 (WindowAttention.forward) and its autograd.  Per window of N <= 64 tokens and
// per head of D = 32, with q, k, v sliced out of one Linear's output [windows, N, 3, heads, D]:
//   S = scale q k^T + bias[head] + mask[window % nW],   P = softmax(S),   O = P v
//   dV = P^T dO,   dP = dO v^T,   dS = P (dP - rowsum(P dP)),   dq = scale dS k,   dk = scale dS^T q,   dbias[head] = sum_windows dS
// A row of S lives in one wave's registers, so the backward takes the softmax again instead of reading statistics or the output: it reads qkv
// and dO and writes dqkv.  A row whose mask leaves nothing (-inf everywhere) has O = 0 and no gradient.
//
// One wave per (window, head).  Products as in window_attn.hip: S^T = K Q^T puts query i = 32 b + (lane & 31) on the lane and keys
// j = 32 a + 8 (e >> 2) + (e & 3) + 4 hh into the accumulators (hh = lane >> 5), so the softmax is in-lane plus one exchange, and P^T is the
// B operand of O^T = V^T P^T as it stands.  The products that sum over queries need the lane to be the key: P and dS cross through LDS.
// Bias and mask come packed in the accumulator layout (sd_window_attn_pack); padded keys carry -inf in the bias.
#include <math.h>

#include "cgd_device.h"

namespace sd {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kPackFloats = 4096;     // sd_window_attn_packed_floats()
constexpr int D = 32;

__device__ __forceinline__ f32x16 mfma(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.f;
    return z;
}
__device__ __forceinline__ int acc_row(int e, int hh) { return 8 * (e >> 2) + (e & 3) + 4 * hh; }

// 16 consecutive elements of row p (half hh of its 32), 0 where there is no such row
template <typename T>
__device__ __forceinline__ void load_half_row(const T *__restrict__ base, long stride, int p, int n, int hh, float mul, float (&o)[16]) {
    constexpr int N = VecIO<T>::N;
    if (p < n) {
        const T *src = base + (size_t)p * stride + 16 * hh;
#pragma unroll
        for (int u = 0; u < 16 / N; ++u) {
            float v[N];
            VecIO<T>::load(src + u * N, v);
#pragma unroll
            for (int i = 0; i < N; ++i) o[u * N + i] = v[i] * mul;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store4(T *p, float x, float y, float z, float w) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(x, y, z, w);
    } else {
        *reinterpret_cast<uint2 *>(p) = make_uint2((unsigned)f32_to_bf16(x) | ((unsigned)f32_to_bf16(y) << 16), (unsigned)f32_to_bf16(z) | ((unsigned)f32_to_bf16(w) << 16));
    }
}
// an accumulator tile whose rows are d and whose column is the lane's token
template <typename T>
__device__ __forceinline__ void store_tile(T *__restrict__ base, long stride, int p, int n, int hh, const f32x16 &o, float mul) {
    if (p >= n) return;
    T *dst = base + (size_t)p * stride + 4 * hh;
#pragma unroll
    for (int g = 0; g < 4; ++g) store4(dst + 8 * g, o[4 * g] * mul, o[4 * g + 1] * mul, o[4 * g + 2] * mul, o[4 * g + 3] * mul);
}

// P^T of query tile b: acc[a] = bias (+ mask) + K Q^T, then its softmax over the keys; probabilities come out normalised
template <int NT>
__device__ __forceinline__ void scores(f32x16 (&acc)[NT], const float (&kf)[NT][16], const float (&qf)[16], const float4 *__restrict__ bias, const float4 *__restrict__ mask,
                                       int b, bool live) {
#pragma unroll
    for (int a = 0; a < NT; ++a) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 v = bias[((a * 2 + b) * 4 + g) * 64];
            acc[a][4 * g] = v.x, acc[a][4 * g + 1] = v.y, acc[a][4 * g + 2] = v.z, acc[a][4 * g + 3] = v.w;
        }
    }
    if (mask) {
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 v = mask[((a * 2 + b) * 4 + g) * 64];
                acc[a][4 * g] += v.x, acc[a][4 * g + 1] += v.y, acc[a][4 * g + 2] += v.z, acc[a][4 * g + 3] += v.w;
            }
    }
#pragma unroll
    for (int s = 0; s < 16; ++s)
#pragma unroll
        for (int a = 0; a < NT; ++a) acc[a] = mfma(kf[a][s], qf[s], acc[a]);
    float m = -INFINITY;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[a][e]);
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    if (m == -INFINITY) m = 0.f;                      // nothing left: every probability is 0
    float l = 0.f;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            acc[a][e] = ex2((acc[a][e] - m) * 1.4426950408889634f);
            l += acc[a][e];
        }
    l += __shfl_xor(l, 32, 64);
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[a][e] = live ? acc[a][e] * inv : 0.f;       // a query row behind the window holds nothing
}

template <typename T, int NT>
__global__ __launch_bounds__(256) void window_train_fwd(const T *__restrict__ qkv, const float *__restrict__ bias_p, const float *__restrict__ mask_p,
                                                        const int *__restrict__ mask_any, T *__restrict__ out, int njobs, int nW, int heads, int N, float scale) {
    const int lane = threadIdx.x & 63, r = lane & 31, hh = lane >> 5;
    const int job = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
    if (job >= njobs) return;
    const int win = job / heads, head = job - win * heads;
    const long C = (long)heads * D, stride = 3 * C;
    const T *q = qkv + (size_t)win * N * stride + (size_t)head * D, *k = q + C, *v = k + C;
    const float4 *bp = reinterpret_cast<const float4 *>(bias_p + (size_t)head * kPackFloats) + lane;
    const float4 *mp = mask_p && mask_any[win % nW] != 0 ? reinterpret_cast<const float4 *>(mask_p + (size_t)(win % nW) * kPackFloats) + lane : nullptr;
    float kf[NT][16], vf[NT][16];
#pragma unroll
    for (int a = 0; a < NT; ++a) {
        load_half_row(k, stride, 32 * a + r, N, hh, 1.f, kf[a]);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int j = 32 * a + acc_row(e, hh);
            vf[a][e] = j < N ? VecIO<T>::load1(v + (size_t)j * stride + r) : 0.f;
        }
    }
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        float qf[16];
        load_half_row(q, stride, 32 * b + r, N, hh, scale, qf);
        f32x16 p[NT];
        scores<NT>(p, kf, qf, bp, mp, b, 32 * b + r < N);
        f32x16 o = zero16();
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int e = 0; e < 16; ++e) o = mfma(vf[a][e], p[a][e], o);
        store_tile(out + (size_t)win * N * C + (size_t)head * D, C, 32 * b + r, N, hh, o, 1.f);
    }
}

// Each wave keeps one head and takes windows slab, slab + slabs, ...: the bias gradient of all of them stays in its accumulators and leaves once,
// as one slab in the packed layout.
template <typename T, int NT>
__global__ __launch_bounds__(256) void window_train_bwd(const T *__restrict__ qkv, const float *__restrict__ bias_p, const float *__restrict__ mask_p,
                                                        const int *__restrict__ mask_any, const T *__restrict__ dout, T *__restrict__ dqkv, float *__restrict__ slabs,
                                                        int windows, int nslab, int nW, int heads, int N, float scale) {
    constexpr int PITCH = 32 * NT + 4;                 // floats per query row: 16-byte rows that start on different banks
    __shared__ __attribute__((aligned(16))) float cross[4][32 * PITCH];
    float *mine = cross[threadIdx.x >> 6];
    const int lane = threadIdx.x & 63, r = lane & 31, hh = lane >> 5;
    const int job = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
    if (job >= nslab * heads) return;                  // whole waves; no workgroup barrier below
    const int slab = job / heads, head = job - slab * heads;
    const long C = (long)heads * D, stride = 3 * C;
    const float4 *bp = reinterpret_cast<const float4 *>(bias_p + (size_t)head * kPackFloats) + lane;
    f32x16 db[NT][NT];
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) db[a][b] = zero16();
    for (int win = slab; win < windows; win += nslab) {
        const T *q = qkv + (size_t)win * N * stride + (size_t)head * D, *k = q + C, *v = k + C;
        const T *go = dout + (size_t)win * N * C + (size_t)head * D;
        T *dq = dqkv + (size_t)win * N * stride + (size_t)head * D, *dk = dq + C, *dv = dk + C;
        const float4 *mp = mask_p && mask_any[win % nW] != 0 ? reinterpret_cast<const float4 *>(mask_p + (size_t)(win % nW) * kPackFloats) + lane : nullptr;
        f32x16 ak[NT], av[NT];
#pragma unroll
        for (int a = 0; a < NT; ++a) ak[a] = av[a] = zero16();
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            f32x16 p[NT], ds[NT];
            {
                float kf[NT][16], qf[16];
#pragma unroll
                for (int a = 0; a < NT; ++a) load_half_row(k, stride, 32 * a + r, N, hh, 1.f, kf[a]);
                load_half_row(q, stride, 32 * b + r, N, hh, scale, qf);
                scores<NT>(p, kf, qf, bp, mp, b, 32 * b + r < N);
            }
            {
                float vf[NT][16], of[16];
#pragma unroll
                for (int a = 0; a < NT; ++a) load_half_row(v, stride, 32 * a + r, N, hh, 1.f, vf[a]);
                load_half_row(go, C, 32 * b + r, N, hh, 1.f, of);
#pragma unroll
                for (int a = 0; a < NT; ++a) {
                    ds[a] = zero16();
#pragma unroll
                    for (int s = 0; s < 16; ++s) ds[a] = mfma(vf[a][s], of[s], ds[a]);
                }
            }
            float dot = 0.f;
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
                for (int e = 0; e < 16; ++e) dot = fmaf(p[a][e], ds[a][e], dot);
            dot += __shfl_xor(dot, 32, 64);
#pragma unroll
            for (int a = 0; a < NT; ++a)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    ds[a][e] = 32 * b + r < N ? p[a][e] * (ds[a][e] - dot) : 0.f;
                    db[a][b][e] += ds[a][e];
                }
            {
                f32x16 aq = zero16();
#pragma unroll
                for (int a = 0; a < NT; ++a)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int j = 32 * a + acc_row(e, hh);
                        aq = mfma(j < N ? VecIO<T>::load1(k + (size_t)j * stride + r) : 0.f, ds[a][e], aq);
                    }
                store_tile(dq, stride, 32 * b + r, N, hh, aq, scale);
            }
            // rows i of tile b of P (then dS) into LDS, columns out: the lane becomes the key.  The image is the wave's own: its LDS operations
            // execute in order, the fences hold the compiler back.
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int a = 0; a < NT; ++a)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x16 &x = which ? ds[a] : p[a];
                        *reinterpret_cast<float4 *>(mine + r * PITCH + 32 * a + 8 * g + 4 * hh) = make_float4(x[4 * g], x[4 * g + 1], x[4 * g + 2], x[4 * g + 3]);
                    }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                const T *src = which ? q : go;
                const long pitch = which ? stride : C;
                float rf[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int i = 32 * b + acc_row(e, hh);
                    rf[e] = i < N ? VecIO<T>::load1(src + (size_t)i * pitch + r) : 0.f;
                }
#pragma unroll
                for (int a = 0; a < NT; ++a)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float x = mine[acc_row(e, hh) * PITCH + 32 * a + r];
                        if (which) ak[a] = mfma(rf[e], x, ak[a]);
                        else av[a] = mfma(rf[e], x, av[a]);
                    }
            }
        }
#pragma unroll
        for (int a = 0; a < NT; ++a) {
            store_tile(dk, stride, 32 * a + r, N, hh, ak[a], scale);
            store_tile(dv, stride, 32 * a + r, N, hh, av[a], 1.f);
        }
    }
    float4 *out = reinterpret_cast<float4 *>(slabs + (size_t)job * (NT * NT * 1024)) + lane;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                out[((a * NT + b) * 4 + g) * 64] = make_float4(db[a][b][4 * g], db[a][b][4 * g + 1], db[a][b][4 * g + 2], db[a][b][4 * g + 3]);
}

// dbias[head][i][j] = the sum of the slabs, in slab order, unpacked
template <int NT>
__global__ __launch_bounds__(256) void window_train_dbias(const float *__restrict__ slabs, float *__restrict__ dbias, int nslab, int heads, int N) {
    const int head = blockIdx.y, at = blockIdx.x * 256 + threadIdx.x;       // at < NT * NT * 1024
    const int c = at & 3, lane = (at >> 2) & 63, g = (at >> 8) & 3, b = (at >> 10) & (NT - 1), a = at >> (NT == 2 ? 11 : 10);
    const int j = 32 * a + 8 * g + c + 4 * (lane >> 5), i = 32 * b + (lane & 31);
    if (i >= N || j >= N) return;
    float s = 0.f;
    for (int w = 0; w < nslab; ++w) s += slabs[((size_t)w * heads + head) * (NT * NT * 1024) + at];
    dbias[((size_t)head * N + i) * N + j] = s;
}

// waves of the backward: about two per SIMD, none without a window
int slabs_for(long windows, int heads) {
    const long want = (2048 + heads - 1) / heads;
    return (int)(want < windows ? want : windows);
}

int check_args(const void *qkv, const float *bias, const float *mask, const int32_t *flags, int dtype, long windows, int mask_windows, int heads, int N, int d) {
    if (!qkv || !bias) return SD_E_NULL;
    if (dtype != SD_F32 && dtype != SD_BF16) return SD_E_DTYPE;
    if (!sd_window_attn_train_supported(N, d)) return SD_E_UNSUPPORTED;
    if (windows <= 0 || heads <= 0 || windows > 0x7ffffff0L / heads || (mask && (!flags || mask_windows <= 0 || windows % mask_windows != 0))) return SD_E_SHAPE;
    if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(mask)) & 15) return SD_E_ALIGN;
    return SD_OK;
}

template <typename T, int NT>
int fwd_launch(const void *qkv, const float *bias, const float *mask, const int32_t *flags, void *out, long windows, int nW, int heads, int N, float scale, hipStream_t st) {
    const int jobs = (int)(windows * heads);
    hipLaunchKernelGGL((window_train_fwd<T, NT>), dim3((unsigned)((jobs + 3) / 4)), dim3(256), 0, st, static_cast<const T *>(qkv), bias, mask, (const int *)flags,
                       static_cast<T *>(out), jobs, nW, heads, N, scale);
    return (int)hipGetLastError();
}
template <typename T, int NT>
int bwd_launch(const void *qkv, const float *bias, const float *mask, const int32_t *flags, const void *dout, void *dqkv, float *dbias, long windows, int nW, int heads,
               int N, float scale, float *slabs, hipStream_t st) {
    const int ns = slabs_for(windows, heads);
    hipLaunchKernelGGL((window_train_bwd<T, NT>), dim3((unsigned)((ns * heads + 3) / 4)), dim3(256), 0, st, static_cast<const T *>(qkv), bias, mask, (const int *)flags,
                       static_cast<const T *>(dout), static_cast<T *>(dqkv), slabs, (int)windows, ns, nW, heads, N, scale);
    hipLaunchKernelGGL((window_train_dbias<NT>), dim3(NT * NT * 4, (unsigned)heads), dim3(256), 0, st, slabs, dbias, ns, heads, N);
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace sd

extern "C" {

int sd_window_attn_train_supported(int tokens_per_window, int head_dim) { return tokens_per_window >= 1 && tokens_per_window <= 64 && head_dim == sd::D; }

int sd_window_attn_train_fwd(const void *qkv, const float *bias_packed, const float *mask_packed, const int32_t *mask_flags, void *out, int dtype, long windows,
                             int mask_windows, int heads, int tokens_per_window, int head_dim, float scale, void *stream) {
    const int rc = sd::check_args(qkv, bias_packed, mask_packed, mask_flags, dtype, windows, mask_windows, heads, tokens_per_window, head_dim);
    if (rc != SD_OK) return rc;
    if (!out) return SD_E_NULL;
    if (reinterpret_cast<uintptr_t>(out) & 15) return SD_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int N = tokens_per_window;
#define SD_FWD(T, NT) sd::fwd_launch<T, NT>(qkv, bias_packed, mask_packed, mask_flags, out, windows, mask_windows, heads, N, scale, st)
    if (dtype == SD_F32) return N <= 32 ? SD_FWD(float, 1) : SD_FWD(float, 2);
    return N <= 32 ? SD_FWD(sd::bf16_t, 1) : SD_FWD(sd::bf16_t, 2);
#undef SD_FWD
}

size_t sd_window_attn_train_workspace_bytes(long windows, int heads, int tokens_per_window) {
    if (windows <= 0 || heads <= 0 || windows > 0x7ffffff0L / heads || tokens_per_window < 1 || tokens_per_window > 64) return 0;
    return (size_t)sd::slabs_for(windows, heads) * heads * (tokens_per_window <= 32 ? 1024 : 4096) * sizeof(float);
}

int sd_window_attn_train_bwd(const void *qkv, const float *bias_packed, const float *mask_packed, const int32_t *mask_flags, const void *dout, void *dqkv, float *dbias,
                             int dtype, long windows, int mask_windows, int heads, int tokens_per_window, int head_dim, float scale, void *workspace,
                             size_t workspace_bytes, void *stream) {
    const int rc = sd::check_args(qkv, bias_packed, mask_packed, mask_flags, dtype, windows, mask_windows, heads, tokens_per_window, head_dim);
    if (rc != SD_OK) return rc;
    if (!dout || !dqkv || !dbias) return SD_E_NULL;
    if (((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dqkv)) & 15) || (reinterpret_cast<uintptr_t>(dbias) & 3)) return SD_E_ALIGN;
    if (!workspace || workspace_bytes < sd_window_attn_train_workspace_bytes(windows, heads, tokens_per_window) || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return SD_E_WORKSPACE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int N = tokens_per_window;
    float *slabs = static_cast<float *>(workspace);
#define SD_BWD(T, NT) sd::bwd_launch<T, NT>(qkv, bias_packed, mask_packed, mask_flags, dout, dqkv, dbias, windows, mask_windows, heads, N, scale, slabs, st)
    if (dtype == SD_F32) return N <= 32 ? SD_BWD(float, 1) : SD_BWD(float, 2);
    return N <= 32 ? SD_BWD(sd::bf16_t, 1) : SD_BWD(sd::bf16_t, 2);
#undef SD_BWD
}

}  // extern "C"
