// window_train.hip -- window multi-head self-attention with a learned bias, forward and backward (a Swin student's blocks), gfx950.
//
// Reference: mmseg/models/backbones/swin_transformer.py:119-153 (WindowAttention.forward) and its autograd.  Per window of N <= 64 tokens and
// per head of D = 32, with q, k, v sliced out of one Linear's output [windows, N, 3, heads, D]:
//   S = scale q k^T + bias[head] + mask[window % nW],   P = softmax(S),   O = P v
//   dV = P^T dO,   dP = dO v^T,   dS = P (dP - rowsum(P dP)),   dq = scale dS k,   dk = scale dS^T q,   dbias[head] = sum_windows dS
// A row of S lives in one wave's registers, so the backward takes the softmax again instead of reading statistics or the output: it reads qkv
// and dO and writes dqkv.  A row whose mask leaves nothing (-inf everywhere) has O = 0 and no gradient.
//
// A workgroup keeps one head and walks over windows; wave w of its NT = ceil(N / 32) waves owns the 32 queries of tile w, then (dV, dK) the 32 keys
// of tile w.  The operands of a window come into LDS as rows, 16 bytes per thread, and the next window's are on their way to registers meanwhile.
// S^T = K Q^T puts query i = 32 w + (lane & 31) on the lane and keys j = 32 a + 8 (e >> 2) + (e & 3) + 4 hh into the accumulators (hh = lane >> 5):
// the softmax is in-lane plus one exchange with the other half-wave, and P^T is the B operand of O^T = V^T P^T as it stands.  The products that sum
// over queries need the lane to be the key: P, then dS, cross through LDS.  The bias gradient of all windows of a workgroup stays in its accumulators
// and leaves once, as one slab; the slabs are joined in slab order.
//   fp32 storage: v_mfma_f32_32x32x2_f32, exact products.
//   bf16 storage: v_mfma_f32_32x32x16_bf16 on the operands as stored.  P and dS enter their products as two bf16 terms (the value and what its
//   rounding left): one term alone would put an error as large as the result's own rounding on every output; the second costs 12 of 32 MFMAs.
//   Softmax, dS and the bias gradient are fp32.  Operand columns come from the row images by transposed LDS reads (ds_read_b64_tr_b16).
#include <math.h>

#include "cgd_device.h"

namespace sd {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
constexpr int D = 32;

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.f;
    return z;
}

// ---- products on LDS images ------------------------------------------------------------------------------------------------------------------
// An image holds rows of 32 elements, PITCH apart (16-byte rows that start on different banks); rows [N, rows(N)) are zero.  The cross image holds one
// row of keys per query.
template <typename T>
struct Lds;

template <>
struct Lds<float> {
    static constexpr int PITCH = 36, CHUNKS = 8;                                  // CHUNKS: 16-byte pieces of a row
    static __host__ __device__ constexpr int rows(int N) { return (N + 7) & ~7; }
    static constexpr int cross_pitch(int NT) { return 32 * NT + 4; }
    static __host__ __device__ constexpr size_t cross_bytes(int N, int NT) { return (size_t)rows(N) * (32 * NT + 4) * 4; }

    typedef f32x16 Operand;                                                       // a tile of P or dS as its products take it
    static __device__ __forceinline__ Operand operand(const f32x16 &p) { return p; }

    // acc[m][n] += sum_d A[32 t + m][d] B[pb][d], lane n holding row pb
    template <int NT>
    static __device__ __forceinline__ void rows_product(f32x16 (&acc)[NT], const float *A, const float *B, int pb, int N, int r, int hh) {
        const int last = rows(N) - 1;                                             // rows behind the image: any finite row, masked by the caller
        const float *b = B + min(pb, last) * PITCH + 16 * hh;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float4 bv = *reinterpret_cast<const float4 *>(b + 4 * u);
#pragma unroll
            for (int a = 0; a < NT; ++a) {
                const float4 av = *reinterpret_cast<const float4 *>(A + min(32 * a + r, last) * PITCH + 16 * hh + 4 * u);
                acc[a] = __builtin_amdgcn_mfma_f32_32x32x2f32(av.x, bv.x, acc[a], 0, 0, 0);
                acc[a] = __builtin_amdgcn_mfma_f32_32x32x2f32(av.y, bv.y, acc[a], 0, 0, 0);
                acc[a] = __builtin_amdgcn_mfma_f32_32x32x2f32(av.z, bv.z, acc[a], 0, 0, 0);
                acc[a] = __builtin_amdgcn_mfma_f32_32x32x2f32(av.w, bv.w, acc[a], 0, 0, 0);
            }
        }
    }
    // acc[d][i] += sum_j M[j][d] p[j][i], p in the accumulator layout
    template <int NT>
    static __device__ __forceinline__ void columns_product(f32x16 &acc, const float *M, const Operand (&p)[NT], int N, int lane) {
        const int r = lane & 31, hh = lane >> 5;
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (32 * a + 8 * g < N) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(M[(32 * a + 8 * g + c + 4 * hh) * PITCH + r], p[a][4 * g + c], acc, 0, 0, 0);
                }
    }
    // the wave's query rows of p into the cross image
    template <int NT>
    static __device__ __forceinline__ void cross_write(float *x, const Operand (&p)[NT], int i, int N, int hh) {
        if (i >= rows(N)) return;
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<float4 *>(x + i * cross_pitch(NT) + 32 * a + 8 * g + 4 * hh) =
                    make_float4(p[a][4 * g], p[a][4 * g + 1], p[a][4 * g + 2], p[a][4 * g + 3]);
    }
    // acc[d][j] += sum_i M[i][d] x[i][j], lane column j = 32 tile + (lane & 31)
    template <int NT>
    static __device__ __forceinline__ void cross_product(f32x16 &acc, const float *M, const float *x, int tile, int N, int lane) {
        const int r = lane & 31, hh = lane >> 5;
        for (int i0 = 0; i0 < N; i0 += 8) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int i = i0 + c + 4 * hh;
                acc = __builtin_amdgcn_mfma_f32_32x32x2f32(M[i * PITCH + r], x[i * cross_pitch(NT) + 32 * tile + r], acc, 0, 0, 0);
            }
        }
    }
};

template <>
struct Lds<bf16_t> {
    static constexpr int PITCH = 40, CHUNKS = 4;
    static __host__ __device__ constexpr int rows(int N) { return (N + 15) & ~15; }
    static constexpr int cross_pitch(int NT) { return 32 * NT + 8; }
    static __host__ __device__ constexpr size_t plane(int N, int NT) { return (size_t)rows(N) * (32 * NT + 8); }       // elements of one of the two terms
    static __host__ __device__ constexpr size_t cross_bytes(int N, int NT) { return 2 * plane(N, NT) * 2; }

    static __device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    // four rows x 16 columns per 16 lanes, delivered by column: lane 16 g + li gets column col0 + 16 g + li of rows row .. row + 3 (then row2 .. row2 + 3)
    static __device__ __forceinline__ bf16x8 columns(const bf16_t *img, int pitch, int row, int row2, int col0, int lane) {
        typedef s16x4 __attribute__((address_space(3))) * lds_p;
        const int li = lane & 15, off = (li >> 2) * pitch + col0 + 16 * ((lane >> 4) & 1) + 4 * (li & 3);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(img + row * pitch + off));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(img + row2 * pitch + off));
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        return __builtin_bit_cast(bf16x8, v);
    }
    template <int NT>
    static __device__ __forceinline__ void rows_product(f32x16 (&acc)[NT], const bf16_t *A, const bf16_t *B, int pb, int N, int r, int hh) {
        const int last = rows(N) - 1;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const bf16x8 bv = *reinterpret_cast<const bf16x8 *>(B + min(pb, last) * PITCH + 16 * t + 8 * hh);
#pragma unroll
            for (int a = 0; a < NT; ++a) acc[a] = mfma(*reinterpret_cast<const bf16x8 *>(A + min(32 * a + r, last) * PITCH + 16 * t + 8 * hh), bv, acc[a]);
        }
    }
    // p = first + second, each bf16, to 2^-17 of p; elements 8 t .. 8 t + 7 of the accumulator tile in first[t], second[t].  On pairs: one conversion
    // instruction takes two values.
    struct Operand {
        bf16x8 first[2], second[2];
    };
    static __device__ __forceinline__ Operand operand(const f32x16 &p) {
        Operand o;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const f32x2 v = {p[e], p[e + 1]};
            const bf16x2 f = __builtin_convertvector(v, bf16x2), s = __builtin_convertvector(v - __builtin_convertvector(f, f32x2), bf16x2);
            o.first[e >> 3][e & 7] = f[0], o.first[e >> 3][(e & 7) + 1] = f[1];
            o.second[e >> 3][e & 7] = s[0], o.second[e >> 3][(e & 7) + 1] = s[1];
        }
        return o;
    }
    template <int NT>
    static __device__ __forceinline__ void columns_product(f32x16 &acc, const bf16_t *M, const Operand (&p)[NT], int N, int lane) {
        const int hh = lane >> 5;
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (32 * a + 16 * t < N) {
                    const int j0 = 32 * a + 16 * t + 4 * hh;                       // accumulator rows 8 t .. 8 t + 7 are j0 .. j0 + 3 and j0 + 8 .. j0 + 11
                    const bf16x8 m = columns(M, PITCH, j0, j0 + 8, 0, lane);
                    acc = mfma(m, p[a].first[t], acc);
                    acc = mfma(m, p[a].second[t], acc);
                }
    }
    template <int NT>
    static __device__ __forceinline__ void cross_write(bf16_t *x, const Operand (&p)[NT], int i, int N, int hh) {
        if (i >= rows(N)) return;
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const u32x4 f = __builtin_bit_cast(u32x4, p[a].first[t]), s = __builtin_bit_cast(u32x4, p[a].second[t]);
                bf16_t *to = x + i * cross_pitch(NT) + 32 * a + 16 * t + 4 * hh;
                *reinterpret_cast<uint2 *>(to) = make_uint2(f[0], f[1]);
                *reinterpret_cast<uint2 *>(to + 8) = make_uint2(f[2], f[3]);
                *reinterpret_cast<uint2 *>(to + plane(N, NT)) = make_uint2(s[0], s[1]);
                *reinterpret_cast<uint2 *>(to + plane(N, NT) + 8) = make_uint2(s[2], s[3]);
            }
    }
    template <int NT>
    static __device__ __forceinline__ void cross_product(f32x16 &acc, const bf16_t *M, const bf16_t *x, int tile, int N, int lane) {
        const int hh = lane >> 5;
        for (int i0 = 0; i0 < N; i0 += 16) {
            const int i = i0 + 8 * hh;
            const bf16x8 m = columns(M, PITCH, i, i + 4, 0, lane);
            acc = mfma(m, columns(x, cross_pitch(NT), i, i + 4, 32 * tile, lane), acc);
            acc = mfma(m, columns(x + plane(N, NT), cross_pitch(NT), i, i + 4, 32 * tile, lane), acc);
        }
    }
};

template <typename T>
__host__ __device__ constexpr size_t image_elems(int N) { return (size_t)Lds<T>::rows(N) * Lds<T>::PITCH; }

// ---- staging -----------------------------------------------------------------------------------------------------------------------------------
// A matrix of N rows of 32 elements, `stride` apart, through registers into an image: NT waves move 64 NT / CHUNKS rows at a time.
template <typename T, int NT>
struct Stage {
    static constexpr int CH = Lds<T>::CHUNKS, STEP = 64 * NT / CH, PASSES = 32 * NT / STEP;
    u32x4 reg[PASSES];
    __device__ __forceinline__ void load(const T *base, long stride, int N) {
        const int row = threadIdx.x / CH, ch = threadIdx.x % CH;
#pragma unroll
        for (int u = 0; u < PASSES; ++u)              // every lane loads, rows behind the window the last one again: a register written in part stays live all along
            reg[u] = *(reinterpret_cast<const u32x4 *>(base + (size_t)min(row + u * STEP, N - 1) * stride) + ch);
    }
    __device__ __forceinline__ void clear() {
        const u32x4 z = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int u = 0; u < PASSES; ++u) reg[u] = z;
    }
    __device__ __forceinline__ void store(T *img, int N) const {
        const int row = threadIdx.x / CH, ch = threadIdx.x % CH;
#pragma unroll
        for (int u = 0; u < PASSES; ++u)
            if (row + u * STEP < N) *(reinterpret_cast<u32x4 *>(img + (row + u * STEP) * Lds<T>::PITCH) + ch) = reg[u];
    }
};
// the zero rows behind an image's last one
template <typename T, int NT>
__device__ __forceinline__ void zero_tail(T *img, int N) {
    const int chunks = (Lds<T>::rows(N) - N) * Lds<T>::CHUNKS;
    for (int u = threadIdx.x; u < chunks; u += 64 * NT) {
        const u32x4 z = {0u, 0u, 0u, 0u};
        *(reinterpret_cast<u32x4 *>(img + (N + u / Lds<T>::CHUNKS) * Lds<T>::PITCH) + u % Lds<T>::CHUNKS) = z;
    }
}

template <typename T>
__device__ __forceinline__ void store4(T *p, float x, float y, float z, float w) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(x, y, z, w);
    } else {
        *reinterpret_cast<uint2 *>(p) =
            make_uint2((unsigned)f32_to_bf16(x) | ((unsigned)f32_to_bf16(y) << 16), (unsigned)f32_to_bf16(z) | ((unsigned)f32_to_bf16(w) << 16));
    }
}
// an accumulator tile whose rows are d and whose column is the lane's token
template <typename T>
__device__ __forceinline__ void store_tile(T *__restrict__ base, long stride, int p, int N, int hh, const f32x16 &o, float mul) {
    if (p >= N) return;
    T *dst = base + (size_t)p * stride + 4 * hh;
#pragma unroll
    for (int g = 0; g < 4; ++g) store4(dst + 8 * g, o[4 * g] * mul, o[4 * g + 1] * mul, o[4 * g + 2] * mul, o[4 * g + 3] * mul);
}

// ---- the softmax of one query tile ---------------------------------------------------------------------------------------------------------------
// p: K Q^T on entry, probabilities on return.  bias / mask: packed tables at (tile, lane).
template <int NT>
__device__ __forceinline__ void softmax_tile(f32x16 (&p)[NT], const float4 *__restrict__ bias, const float4 *__restrict__ mask, float scale, bool live) {
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 v = bias[(a * NT * 4 + g) * 64];
            p[a][4 * g] = fmaf(p[a][4 * g], scale, v.x), p[a][4 * g + 1] = fmaf(p[a][4 * g + 1], scale, v.y);
            p[a][4 * g + 2] = fmaf(p[a][4 * g + 2], scale, v.z), p[a][4 * g + 3] = fmaf(p[a][4 * g + 3], scale, v.w);
        }
    if (mask) {
#pragma unroll
        for (int a = 0; a < NT; ++a)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 v = mask[(a * NT * 4 + g) * 64];
                p[a][4 * g] += v.x, p[a][4 * g + 1] += v.y, p[a][4 * g + 2] += v.z, p[a][4 * g + 3] += v.w;
            }
    }
    float m = -INFINITY;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, p[a][e]);
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    if (m == -INFINITY) m = 0.f;                      // nothing left: every probability is 0
    float l = 0.f;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            p[a][e] = ex2((p[a][e] - m) * 1.4426950408889634f);
            l += p[a][e];
        }
    l += __shfl_xor(l, 32, 64);
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) p[a][e] = live ? p[a][e] * inv : 0.f;        // a query row behind the window holds nothing
}

// ---- tables --------------------------------------------------------------------------------------------------------------------------------------
// bias [heads][N][N], then mask [nW][N][N], into the accumulator layout [a][b][e >> 2][lane][e & 3]: padded keys -inf in the bias and 0 in the mask,
// padded queries 0; any[w] = the mask of window w has a nonzero entry
template <int NT>
__global__ __launch_bounds__(256) void window_tables(const float *__restrict__ bias, const float *__restrict__ mask, float *__restrict__ packed, int *__restrict__ any,
                                                     int heads, int N) {
    const int t = blockIdx.x;
    const float *src = t < heads ? bias + (size_t)t * N * N : mask + (size_t)(t - heads) * N * N;
    const float pad = t < heads ? -INFINITY : 0.f;
    int nonzero = 0;
    for (int at = threadIdx.x; at < NT * NT * 1024; at += 256) {
        const int c = at & 3, lane = (at >> 2) & 63, g = (at >> 8) & 3, ab = at >> 10, b = ab % NT, a = ab / NT;
        const int j = 32 * a + 8 * g + c + 4 * (lane >> 5), i = 32 * b + (lane & 31);
        const float v = j >= N ? pad : (i < N ? src[(size_t)i * N + j] : 0.f);
        packed[(size_t)t * (NT * NT * 1024) + at] = v;
        nonzero |= v != 0.f;
    }
    nonzero = __syncthreads_or(nonzero);
    if (t >= heads && threadIdx.x == 0) any[t - heads] = nonzero;
}

// Workgroups that share windows -- neighbouring heads, whose rows share cache lines -- sit on one of the eight chiplets: consecutive logical ids do.
__device__ __forceinline__ int logical_block() {
    const int n = gridDim.x, id = blockIdx.x, q = n / 8, rem = n % 8, x = id % 8;
    return (x < rem ? x * (q + 1) : rem * (q + 1) + (x - rem) * q) + id / 8;
}

template <typename T, int NT>
__global__ __launch_bounds__(64 * NT) __attribute__((amdgpu_waves_per_eu(3))) void window_train_fwd(const T *__restrict__ qkv, const float *__restrict__ packed, const int *__restrict__ any, T *__restrict__ out,
                                                            int windows, int nslab, int nW, int heads, int N, float scale) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const size_t img = image_elems<T>(N);
    T *Q = reinterpret_cast<T *>(lds), *K = Q + img, *V = K + img;
    const int lane = threadIdx.x & 63, r = lane & 31, hh = lane >> 5, w = threadIdx.x >> 6;
    const int job = logical_block(), slab = job / heads, head = job - slab * heads;
    const long C = (long)heads * D, stride = 3 * C, wstride = N * stride;
    const T *base = qkv + (size_t)head * D;
    const float4 *bias = reinterpret_cast<const float4 *>(packed + (size_t)head * (NT * NT * 1024)) + w * 256 + lane;
    Stage<T, NT> sq, sk, sv;
    auto fetch = [&](int win) {
        const T *q = base + (size_t)win * wstride;
        sq.load(q, stride, N), sk.load(q + C, stride, N), sv.load(q + 2 * C, stride, N);
    };
    auto none = [&]() { sq.clear(), sk.clear(), sv.clear(); };          // a value on both ways: else the old one would stay live through the loop
    fetch(slab);
    zero_tail<T, NT>(Q, N), zero_tail<T, NT>(K, N), zero_tail<T, NT>(V, N);
    for (int win = slab; win < windows; win += nslab) {
        __syncthreads();                               // the previous window's images are read
        sq.store(Q, N), sk.store(K, N), sv.store(V, N);
        __syncthreads();
        const float4 *mask = nW && any[win % nW] ? reinterpret_cast<const float4 *>(packed + (size_t)(heads + win % nW) * (NT * NT * 1024)) + w * 256 + lane : nullptr;
        f32x16 p[NT], o = zero16();
#pragma unroll
        for (int a = 0; a < NT; ++a) p[a] = zero16();
        Lds<T>::template rows_product<NT>(p, K, Q, 32 * w + r, N, r, hh);
        softmax_tile<NT>(p, bias, mask, scale, 32 * w + r < N);
        win + nslab < windows ? fetch(win + nslab) : none();          // (not before: the registers are the scores' until here)
        typename Lds<T>::Operand po[NT];
#pragma unroll
        for (int a = 0; a < NT; ++a) po[a] = Lds<T>::operand(p[a]);
        Lds<T>::template columns_product<NT>(o, V, po, N, lane);
        store_tile(out + (size_t)win * N * C + (size_t)head * D, C, 32 * w + r, N, hh, o, 1.f);
    }
}

constexpr int kBwdWaves = 2;           // waves per SIMD that the backward's registers leave room for (three: 73 spilled, bf16 76 -> 145 us)

template <typename T, int NT>
__global__ __launch_bounds__(64 * NT, kBwdWaves) void window_train_bwd(const T *__restrict__ qkv, const float *__restrict__ packed, const int *__restrict__ any,
                                                            const T *__restrict__ dout, T *__restrict__ dqkv, float *__restrict__ slabs, int windows, int nslab, int nW,
                                                            int heads, int N, float scale) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const size_t img = image_elems<T>(N);
    T *Q = reinterpret_cast<T *>(lds), *G = Q + img, *K = G + img, *V = K + img, *X = K;          // P and dS cross where K and V were
    const int lane = threadIdx.x & 63, r = lane & 31, hh = lane >> 5, w = threadIdx.x >> 6, i = 32 * w + r;
    const int job = logical_block(), slab = job / heads, head = job - slab * heads;
    const long C = (long)heads * D, stride = 3 * C, wstride = N * stride;
    const T *base = qkv + (size_t)head * D, *gbase = dout + (size_t)head * D;
    const float4 *bias = reinterpret_cast<const float4 *>(packed + (size_t)head * (NT * NT * 1024)) + w * 256 + lane;
    Stage<T, NT> sq, sk, sv, sg;
    auto fetch = [&](int win) {
        const T *q = base + (size_t)win * wstride;
        sq.load(q, stride, N), sk.load(q + C, stride, N), sv.load(q + 2 * C, stride, N);
        sg.load(gbase + (size_t)win * N * C, C, N);
    };
    auto none = [&]() { sq.clear(), sk.clear(), sv.clear(), sg.clear(); };          // a value on both ways: else the old one would stay live through the loop
    fetch(slab);
    zero_tail<T, NT>(Q, N), zero_tail<T, NT>(G, N);
    f32x16 db[NT];
#pragma unroll
    for (int a = 0; a < NT; ++a) db[a] = zero16();
    for (int win = slab; win < windows; win += nslab) {
        __syncthreads();                               // the previous window's images are read
        sq.store(Q, N), sk.store(K, N), sv.store(V, N), sg.store(G, N);
        zero_tail<T, NT>(K, N), zero_tail<T, NT>(V, N);
        __syncthreads();
        const float4 *mask = nW && any[win % nW] ? reinterpret_cast<const float4 *>(packed + (size_t)(heads + win % nW) * (NT * NT * 1024)) + w * 256 + lane : nullptr;
        T *dq = dqkv + (size_t)win * wstride + (size_t)head * D;
        f32x16 p[NT], ds[NT];
#pragma unroll
        for (int a = 0; a < NT; ++a) p[a] = ds[a] = zero16();
        Lds<T>::template rows_product<NT>(p, K, Q, i, N, r, hh);
        softmax_tile<NT>(p, bias, mask, scale, i < N);
        Lds<T>::template rows_product<NT>(ds, V, G, i, N, r, hh);
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
                ds[a][e] = i < N ? p[a][e] * (ds[a][e] - dot) : 0.f;
                db[a][e] += ds[a][e];
            }
        typename Lds<T>::Operand po[NT], so[NT];
#pragma unroll
        for (int a = 0; a < NT; ++a) po[a] = Lds<T>::operand(p[a]), so[a] = Lds<T>::operand(ds[a]);
        {
            f32x16 o = zero16();
            Lds<T>::template columns_product<NT>(o, K, so, N, lane);
            store_tile(dq, stride, i, N, hh, o, scale);
        }
        __syncthreads();                               // K and V are read
        Lds<T>::template cross_write<NT>(X, po, i, N, hh);
        __syncthreads();                               // every query row of P is there
        win + nslab < windows ? fetch(win + nslab) : none();          // (not before: the registers are the scores' and P's until here)
        {
            f32x16 o = zero16();
            Lds<T>::template cross_product<NT>(o, G, X, w, N, lane);
            store_tile(dq + 2 * C, stride, i, N, hh, o, 1.f);
        }
        __syncthreads();                               // P is read
        Lds<T>::template cross_write<NT>(X, so, i, N, hh);
        __syncthreads();
        {
            f32x16 o = zero16();
            Lds<T>::template cross_product<NT>(o, Q, X, w, N, lane);
            store_tile(dq + C, stride, i, N, hh, o, scale);
        }
    }
    float4 *to = reinterpret_cast<float4 *>(slabs + (size_t)job * (NT * NT * 1024)) + w * 256 + lane;
#pragma unroll
    for (int a = 0; a < NT; ++a)
#pragma unroll
        for (int g = 0; g < 4; ++g) to[(a * NT * 4 + g) * 64] = make_float4(db[a][4 * g], db[a][4 * g + 1], db[a][4 * g + 2], db[a][4 * g + 3]);
}

// dbias[head][i][j] = the sum of the slabs, unpacked.  Sixteen waves take every sixteenth slab of the same 64 float4 each; their sums join in wave order.
template <int NT>
__global__ __launch_bounds__(1024) void window_train_dbias(const float *__restrict__ slabs, float *__restrict__ dbias, int nslab, int heads, int N) {
    __shared__ float4 part[16][64];
    const int head = blockIdx.y, lane = threadIdx.x & 63, wv = threadIdx.x >> 6, at = blockIdx.x * 64 + lane;      // float4 number at of the table
    const float4 *src = reinterpret_cast<const float4 *>(slabs) + (size_t)head * (NT * NT * 256) + at;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = wv; k < nslab; k += 16) {
        const float4 v = src[(size_t)k * heads * (NT * NT * 256)];
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    part[wv][lane] = s;
    __syncthreads();
    if (wv) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) {
        const float4 v = part[k][lane];
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    const int l = at & 63, g = (at >> 6) & 3, ab = at >> 8, b = ab % NT, a = ab / NT;
    const int j = 32 * a + 8 * g + 4 * (l >> 5), i = 32 * b + (l & 31);
    if (i >= N) return;
    float *to = dbias + ((size_t)head * N + i) * N + j;
    if (j < N) to[0] = s.x;
    if (j + 1 < N) to[1] = s.y;
    if (j + 2 < N) to[2] = s.z;
    if (j + 3 < N) to[3] = s.w;
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------------------
// Workgroups of a pass: as many as fit the 256 CUs at once (`per_cu`, by LDS), each with the same number of windows but for the last ones.
int slabs_for(long windows, int heads, int per_cu) {
    const long per = (windows * heads + 256L * per_cu - 1) / (256L * per_cu);
    return (int)((windows + per - 1) / per);
}
template <typename T>
size_t fwd_lds(int N) { return 3 * image_elems<T>(N) * sizeof(T); }
template <typename T>
size_t bwd_lds(int N) {
    const size_t two = 2 * image_elems<T>(N) * sizeof(T), cross = Lds<T>::cross_bytes(N, N <= 32 ? 1 : 2);
    return two + (two > cross ? two : cross);
}
int per_cu(size_t lds, int most) {
    const int n = (int)(160 * 1024 / (lds + 512));
    return n < most ? n : most;
}
template <typename T>
int bwd_slabs(long windows, int heads, int N) { return slabs_for(windows, heads, per_cu(bwd_lds<T>(N), kBwdWaves * (N <= 32 ? 4 : 2))); }

bool shape_ok(long windows, int heads, int N) { return windows > 0 && heads > 0 && heads <= 65535 && windows <= 0x3fffffffL / heads && N >= 1 && N <= 64; }
size_t table_floats(int heads, int nW, int N) { return (size_t)(heads + nW) * (N <= 32 ? 1024 : 4096); }

int check_args(const void *qkv, const float *packed, size_t packed_floats, int dtype, long windows, int nW, int heads, int N, int d) {
    if (!qkv || !packed) return SD_E_NULL;
    if (dtype != SD_F32 && dtype != SD_BF16) return SD_E_DTYPE;
    if (!sd_window_attn_train_supported(N, d)) return SD_E_UNSUPPORTED;
    if (!shape_ok(windows, heads, N) || nW < 0 || (nW > 0 && windows % nW != 0)) return SD_E_SHAPE;
    if (packed_floats < sd_window_attn_train_packed_floats(heads, nW, N)) return SD_E_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(packed)) & 15) return SD_E_ALIGN;
    return SD_OK;
}

template <typename T, int NT>
int fwd_launch(const void *qkv, const float *bias, const float *mask, float *packed, void *out, long windows, int nW, int heads, int N, float scale, hipStream_t st) {
    int *any = reinterpret_cast<int *>(packed + table_floats(heads, nW, N));
    hipLaunchKernelGGL((window_tables<NT>), dim3((unsigned)(heads + nW)), dim3(256), 0, st, bias, mask, packed, any, heads, N);
    const size_t lds = fwd_lds<T>(N);
    const int ns = slabs_for(windows, heads, per_cu(lds, N <= 32 ? 12 : 6));
    hipLaunchKernelGGL((window_train_fwd<T, NT>), dim3((unsigned)(ns * heads)), dim3(64 * NT), lds, st, static_cast<const T *>(qkv), packed, any, static_cast<T *>(out),
                       (int)windows, ns, nW, heads, N, scale);
    return (int)hipGetLastError();
}
template <typename T, int NT>
int bwd_launch(const void *qkv, const float *packed, const void *dout, void *dqkv, float *dbias, long windows, int nW, int heads, int N, float scale, float *slabs,
               hipStream_t st) {
    const int *any = reinterpret_cast<const int *>(packed + table_floats(heads, nW, N));
    const int ns = bwd_slabs<T>(windows, heads, N);
    hipLaunchKernelGGL((window_train_bwd<T, NT>), dim3((unsigned)(ns * heads)), dim3(64 * NT), bwd_lds<T>(N), st, static_cast<const T *>(qkv), packed, any,
                       static_cast<const T *>(dout), static_cast<T *>(dqkv), slabs, (int)windows, ns, nW, heads, N, scale);
    hipLaunchKernelGGL((window_train_dbias<NT>), dim3(NT * NT * 4, (unsigned)heads), dim3(1024), 0, st, slabs, dbias, ns, heads, N);
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace sd

extern "C" {

int sd_window_attn_train_supported(int tokens_per_window, int head_dim) { return tokens_per_window >= 1 && tokens_per_window <= 64 && head_dim == sd::D; }

size_t sd_window_attn_train_packed_floats(int heads, int mask_windows, int tokens_per_window) {
    if (heads <= 0 || mask_windows < 0 || tokens_per_window < 1 || tokens_per_window > 64) return 0;
    return sd::table_floats(heads, mask_windows, tokens_per_window) + (size_t)mask_windows;
}

int sd_window_attn_train_fwd(const void *qkv, const float *bias, const float *mask, float *packed, size_t packed_floats, void *out, int dtype, long windows,
                             int mask_windows, int heads, int tokens_per_window, int head_dim, float scale, void *stream) {
    const int rc = sd::check_args(qkv, packed, packed_floats, dtype, windows, mask_windows, heads, tokens_per_window, head_dim);
    if (rc != SD_OK) return rc;
    if (!out || !bias || (mask_windows > 0 && !mask)) return SD_E_NULL;
    if ((reinterpret_cast<uintptr_t>(out) & 15) || ((reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(mask)) & 3)) return SD_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int N = tokens_per_window;
#define SD_FWD(T, NT) sd::fwd_launch<T, NT>(qkv, bias, mask, packed, out, windows, mask_windows, heads, N, scale, st)
    if (dtype == SD_F32) return N <= 32 ? SD_FWD(float, 1) : SD_FWD(float, 2);
    return N <= 32 ? SD_FWD(sd::bf16_t, 1) : SD_FWD(sd::bf16_t, 2);
#undef SD_FWD
}

size_t sd_window_attn_train_workspace_bytes(int dtype, long windows, int heads, int tokens_per_window) {
    if (!sd::shape_ok(windows, heads, tokens_per_window) || (dtype != SD_F32 && dtype != SD_BF16)) return 0;
    const int N = tokens_per_window, ns = dtype == SD_F32 ? sd::bwd_slabs<float>(windows, heads, N) : sd::bwd_slabs<sd::bf16_t>(windows, heads, N);
    return (size_t)ns * heads * (N <= 32 ? 1024 : 4096) * sizeof(float);
}

int sd_window_attn_train_bwd(const void *qkv, const float *packed, size_t packed_floats, const void *dout, void *dqkv, float *dbias, int dtype, long windows,
                             int mask_windows, int heads, int tokens_per_window, int head_dim, float scale, void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = sd::check_args(qkv, packed, packed_floats, dtype, windows, mask_windows, heads, tokens_per_window, head_dim);
    if (rc != SD_OK) return rc;
    if (!dout || !dqkv || !dbias) return SD_E_NULL;
    if (((reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dqkv)) & 15) || (reinterpret_cast<uintptr_t>(dbias) & 3)) return SD_E_ALIGN;
    if (!workspace || workspace_bytes < sd_window_attn_train_workspace_bytes(dtype, windows, heads, tokens_per_window) || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return SD_E_WORKSPACE;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int N = tokens_per_window;
    float *slabs = static_cast<float *>(workspace);
#define SD_BWD(T, NT) sd::bwd_launch<T, NT>(qkv, packed, dout, dqkv, dbias, windows, mask_windows, heads, N, scale, slabs, st)
    if (dtype == SD_F32) return N <= 32 ? SD_BWD(float, 1) : SD_BWD(float, 2);
    return N <= 32 ? SD_BWD(sd::bf16_t, 1) : SD_BWD(sd::bf16_t, 2);
#undef SD_BWD
}

}  // extern "C"
