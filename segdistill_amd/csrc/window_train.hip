// window_train.hip -- window multi-head self-attention with a learned bias, forward and backward (a Swin student's blocks), gfx950.
//
// Reference: mmseg/models/backbones/swin_transformer.py:119-153 (WindowAttention.forward) and its autograd.  Per window of N <= 64 tokens and
// per head of D = 32, with q, k, v sliced out of one Linear's output [windows, N, 3, heads, D]:
//   S = scale q k^T + bias[head] + mask[window % nW],   P = softmax(S),   O = P v
//   dV = P^T dO,   dP = dO v^T,   dS = P (dP - rowsum(P dP)),   dq = scale dS k,   dk = scale dS^T q,   dbias[head] = sum_windows dS
// A row of S lives in one wave's registers, so the backward takes the softmax again instead of reading statistics or the output: it reads qkv
// and dO and writes dqkv.  A row whose mask leaves nothing (-inf everywhere) has O = 0 and no gradient.
//
// A workgroup keeps one head and walks over windows; wave w of its NA = ceil(N / 16) waves owns the 16 queries of tile w, then (dV, dK) the 16 keys
// of tile w.  The operands of a window come into LDS as rows, 16 bytes per thread, and the next window's are on their way to registers meanwhile.
// S^T = K Q^T puts query i = 16 w + (lane & 15) on the lane and its keys into the accumulators: keys 16 a + 4 q + e of the lanes q = lane >> 4 in
// accumulator e of tile a.  A last tile that is not full takes the rows of K in another order (spread), keys 16 a + 4 e + q: the keys it lacks are then
// whole accumulators, NS = ceil(N / 4) hold keys, and NS is known to the compiler (13 of 16 for 7 x 7 windows).  The softmax is in-lane plus two exchanges,
// and P^T is the B operand of O^T = V^T P^T as it stands.  The products that sum over queries need the lane to be the key: P, then dS,
// cross through LDS.  The bias gradient of all windows of a workgroup stays in its accumulators and leaves once, as one slab; the slabs are joined in
// slab order.
//   fp32 storage: v_mfma_f32_16x16x4_f32, exact products.
//   bf16 storage: v_mfma_f32_16x16x32_bf16 on the operands as stored.  P and dS enter their products as two bf16 terms (the
//   value and what its rounding left): one term alone would put an error as large as the result's own rounding on every output.
//   Softmax, dS and the bias gradient are fp32.  Operand columns come from the row images by transposed LDS reads (ds_read_b64_tr_b16).
//
// 2888 windows of 49 tokens, 3 heads, 361 masks (217 MB forward, 380 MB backward in fp32):  fp32 tables 4.7 us, forward 59 (3.7 TB/s; matrix pipe 45 % busy),
// backward 126 to 138 (2.8 to 3.0 TB/s; matrix pipe 52 % busy, tiles of 16 make 64 x 64 of 49 x 49; without HBM traffic it takes 122, without products 77),
// join 5.  bf16: forward 24 (4.6 TB/s), backward 54 (3.5 TB/s; VALU 37 %, LDS 36 % busy and 12 % more in conflicts; without products 43).  Tiles of 32, two waves
// to a window: 75 + 145 and 26.5 + 66; raised wave priority around the products and LDS reads pinned ahead of them: level.
// 2048 windows of 64 tokens, 3 heads, 256 masks (201 and 352 MB in fp32): fp32 53 + 96 us (3.8 and 3.7 TB/s), bf16 30 + 41 (3.4 and 4.3 TB/s).
#include <math.h>

#include <type_traits>

#include "cgd_device.h"

namespace sd {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
constexpr int D = 32;
constexpr f32x4 kZero4 = {0.f, 0.f, 0.f, 0.f};

// ---- products on LDS images ------------------------------------------------------------------------------------------------------------------
// An image holds 16 NA rows of 32 elements, PITCH apart (16-byte pieces of 16 rows cover the banks); rows behind the window are zero.  The cross image
// holds one row of keys per query, a tile's keys in the order of the accumulators.  r = lane & 15, q = lane >> 4.  Sums over tokens take them in the order of
// the accumulators, too: token_of(q, e, spread) of tile a in step 4 a + e.
constexpr int tiles_of(int NS) { return (NS + 3) / 4; }
__host__ __device__ constexpr bool spread_tile(int a, int NS) { return a == NS / 4; }            // the tile that is not full, if there is one
__device__ __forceinline__ int token_of(int q, int e, bool spread) { return spread ? 4 * e + q : 4 * q + e; }
__device__ __forceinline__ int token_of_row(int r, bool spread) { return token_of(r >> 2, r & 3, spread); }      // the tile's row r holds accumulator r & 3 of q = r >> 2
template <typename T>
struct Lds;

template <>
struct Lds<float> {
    static constexpr int PITCH = 36, CHUNKS = 8;                                  // CHUNKS: 16-byte pieces of a row
    static __device__ __forceinline__ int chunk(int, int ch) { return ch; }
    static __host__ __device__ constexpr int cross_pitch(int NA) { return 16 * NA + 4; }          // 16 columns of every fourth row cover the banks, as those of an image
    static __host__ __device__ constexpr size_t cross_bytes(int NA) { return (size_t)16 * NA * cross_pitch(NA) * 4; }

    template <int NA>
    struct Operand {                                                              // the wave's tiles of P or dS as their products take them
        f32x4 v[NA];
    };
    template <int NA>
    static __device__ __forceinline__ Operand<NA> operand(const f32x4 (&p)[NA]) {
        Operand<NA> o;
#pragma unroll
        for (int a = 0; a < NA; ++a) o.v[a] = p[a];
        return o;
    }
    // acc[a][m][n] += sum_d A[16 a + token_of_row(m)][d] B[16 w + n][d]
    template <int NS, int NA = tiles_of(NS)>
    static __device__ __forceinline__ void rows_product(f32x4 (&acc)[NA], const float *A, const float *B, int w, int lane) {
        const int r = lane & 15, d = 8 * (lane >> 4);
        const float *full = A + r * PITCH + d, *part = A + token_of_row(r, true) * PITCH + d, *pb = B + (16 * w + r) * PITCH + d;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const f32x4 bv = *reinterpret_cast<const f32x4 *>(pb + 4 * u);
            f32x4 av[NA];
#pragma unroll
            for (int a = 0; a < NA; ++a) av[a] = *reinterpret_cast<const f32x4 *>((spread_tile(a, NS) ? part : full) + 16 * a * PITCH + 4 * u);
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int a = 0; a < NA; ++a) acc[a] = __builtin_amdgcn_mfma_f32_16x16x4f32(av[a][c], bv[c], acc[a], 0, 0, 0);
        }
    }
    // acc[h][d][i] += sum_j M[j][16 h + d] p[j][i]
    template <int NS>
    static __device__ __forceinline__ void columns_product(f32x4 (&acc)[2], const float *M, const Operand<tiles_of(NS)> &p, int lane) {
        const int q = lane >> 4, r = lane & 15;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const float *m = M + (16 * (s >> 2) + token_of(q, s & 3, spread_tile(s >> 2, NS))) * PITCH + r;
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(m[16 * h], p.v[s >> 2][s & 3], acc[h], 0, 0, 0);
        }
    }
    // the wave's query rows of p into the cross image
    template <int NA>
    static __device__ __forceinline__ void cross_write(float *x, const Operand<NA> &p, int w, int lane) {
        float *to = x + (16 * w + (lane & 15)) * cross_pitch(NA) + 4 * (lane >> 4);
#pragma unroll
        for (int a = 0; a < NA; ++a) *reinterpret_cast<f32x4 *>(to + 16 * a) = p.v[a];
    }
    // acc[h][d][n] += sum_i M[i][16 h + d] x[i][16 w + n]
    template <int NS>
    static __device__ __forceinline__ void cross_product(f32x4 (&acc)[2], const float *M, const float *x, int w, int lane) {
        constexpr int pitch = cross_pitch(tiles_of(NS));
        const int q = lane >> 4, r = lane & 15;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int i = 16 * (s >> 2) + token_of(q, s & 3, spread_tile(s >> 2, NS));
            const float bv = x[i * pitch + 16 * w + r];
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(M[i * PITCH + 16 * h + r], bv, acc[h], 0, 0, 0);
        }
    }
};

template <>
struct Lds<bf16_t> {
    // Rows are an odd number of eight banks apart, so that the 32 lanes of a transposed read (four rows x 16 columns for each 16 of them) meet every bank
    // once; rows 8 .. 15 of a tile have neighbouring 16-byte pieces exchanged, so that 16 rows do where they are read or written by rows.
    static constexpr int PITCH = 48, CHUNKS = 4;
    static __device__ __forceinline__ int chunk(int row, int ch) { return ch ^ ((row >> 3) & 1); }
    static __host__ __device__ constexpr int cross_pitch(int NA) { return NA == 1 ? 16 : NA == 4 ? 80 : 48; }
    static __host__ __device__ constexpr size_t plane(int NA) { return (size_t)16 * NA * cross_pitch(NA); }       // elements of one of the two terms
    static __host__ __device__ constexpr size_t cross_bytes(int NA) { return 2 * plane(NA) * 2; }

    // four rows x 16 columns per 16 lanes, delivered by column: lane 16 q + r gets column r of the four tokens that the lanes q hold
    static __device__ __forceinline__ s16x4 columns(const bf16_t *tile, int pitch, bool spread, int lane) {
        typedef s16x4 __attribute__((address_space(3))) * lds_p;
        const int row = token_of(lane >> 4, (lane >> 2) & 3, spread);
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(tile + row * pitch + 8 * chunk(row, (lane >> 1) & 1) + 4 * (lane & 1)));
    }
    static __device__ __forceinline__ bf16x8 join(s16x4 lo, s16x4 hi) {
        const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        return __builtin_bit_cast(bf16x8, v);
    }
    // An odd last tile goes with a zero one.  (Not by the 16-deep form: hipcc lets it follow the 32-deep one on the same accumulator without the wait that
    // their different lengths need, and its first rows come out wrong.)
    static __device__ __forceinline__ f32x4 mfma32(s16x4 a0, s16x4 a1, s16x4 b0, s16x4 b1, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(join(a0, a1), join(b0, b1), c, 0, 0, 0);
    }

    // p = first + second, each bf16, to 2^-17 of p.  On pairs: one conversion instruction takes two values.
    template <int NA>
    struct Operand {
        s16x4 first[NA], second[NA];
    };
    template <int NA>
    static __device__ __forceinline__ Operand<NA> operand(const f32x4 (&p)[NA]) {
        Operand<NA> o;
#pragma unroll
        for (int a = 0; a < NA; ++a) {
            bf16x4 f, s;
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const f32x2 v = {p[a][e], p[a][e + 1]};
                const bf16x2 f2 = __builtin_convertvector(v, bf16x2), s2 = __builtin_convertvector(v - __builtin_convertvector(f2, f32x2), bf16x2);
                f[e] = f2[0], f[e + 1] = f2[1];
                s[e] = s2[0], s[e + 1] = s2[1];
            }
            o.first[a] = __builtin_bit_cast(s16x4, f);
            o.second[a] = __builtin_bit_cast(s16x4, s);
        }
        return o;
    }
    template <int NS, int NA = tiles_of(NS)>
    static __device__ __forceinline__ void rows_product(f32x4 (&acc)[NA], const bf16_t *A, const bf16_t *B, int w, int lane) {
        const int r = lane & 15, q = lane >> 4;
        const bf16x8 bv = *reinterpret_cast<const bf16x8 *>(B + (16 * w + r) * PITCH + 8 * chunk(r, q));
#pragma unroll
        for (int a = 0; a < NA; ++a) {
            const int row = token_of_row(r, spread_tile(a, NS));
            acc[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8 *>(A + (16 * a + row) * PITCH + 8 * chunk(row, q)), bv, acc[a], 0, 0, 0);
        }
    }
    template <int NA>
    static __device__ __forceinline__ void product(f32x4 &acc, const s16x4 (&m)[NA], const Operand<NA> &p) {
#pragma unroll
        for (int a = 0; a < NA; a += 2) {
            const s16x4 zero = {0, 0, 0, 0};
            const bool pair = a + 1 < NA;
            const int b = pair ? a + 1 : a;
            acc = mfma32(m[a], pair ? m[b] : zero, p.first[a], pair ? p.first[b] : zero, acc);
            acc = mfma32(m[a], pair ? m[b] : zero, p.second[a], pair ? p.second[b] : zero, acc);
        }
    }
    template <int NS, int NA = tiles_of(NS)>
    static __device__ __forceinline__ void columns_product(f32x4 (&acc)[2], const bf16_t *M, const Operand<NA> &p, int lane) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s16x4 m[NA];
#pragma unroll
            for (int a = 0; a < NA; ++a) m[a] = columns(M + 16 * a * PITCH + 16 * h, PITCH, spread_tile(a, NS), lane);
            product<NA>(acc[h], m, p);
        }
    }
    template <int NA>
    static __device__ __forceinline__ void cross_write(bf16_t *x, const Operand<NA> &p, int w, int lane) {
        const int r = lane & 15;
        bf16_t *to = x + (16 * w + r) * cross_pitch(NA) + 8 * chunk(r, lane >> 5) + 4 * ((lane >> 4) & 1);
#pragma unroll
        for (int a = 0; a < NA; ++a) {
            *reinterpret_cast<s16x4 *>(to + 16 * a) = p.first[a];
            *reinterpret_cast<s16x4 *>(to + plane(NA) + 16 * a) = p.second[a];
        }
    }
    template <int NS, int NA = tiles_of(NS)>
    static __device__ __forceinline__ void cross_product(f32x4 (&acc)[2], const bf16_t *M, const bf16_t *x, int w, int lane) {
        Operand<NA> p;
#pragma unroll
        for (int a = 0; a < NA; ++a) {
            const bf16_t *from = x + 16 * a * cross_pitch(NA) + 16 * w;
            p.first[a] = columns(from, cross_pitch(NA), false, lane);
            p.second[a] = columns(from + plane(NA), cross_pitch(NA), false, lane);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            s16x4 m[NA];
#pragma unroll
            for (int a = 0; a < NA; ++a) m[a] = columns(M + 16 * a * PITCH + 16 * h, PITCH, false, lane);
            product<NA>(acc[h], m, p);
        }
    }
};

template <typename T>
__host__ __device__ constexpr size_t image_elems(int NA) { return (size_t)16 * NA * Lds<T>::PITCH; }

// ---- staging -----------------------------------------------------------------------------------------------------------------------------------
// A matrix of N rows of 32 elements, `stride` apart, through registers into an image: NA waves move 64 NA / CHUNKS rows at a time.
template <typename T, int NA>
struct Stage {
    static constexpr int CH = Lds<T>::CHUNKS, STEP = 64 * NA / CH, PASSES = 16 * NA / STEP;
    u32x4 reg[PASSES];
    // `base` is the workgroup's, the lane adds a 32-bit offset (64 rows of 3 * 65535 heads * 128 bytes stay below 2^31)
    __device__ __forceinline__ void load(const T *base, unsigned stride, int N) {
        const unsigned row = threadIdx.x / CH, ch = threadIdx.x % CH;
        const char *from = reinterpret_cast<const char *>(base);
#pragma unroll
        for (int u = 0; u < PASSES; ++u)              // every lane loads, rows behind the window the last one again: a register written in part stays live all along
            reg[u] = *reinterpret_cast<const u32x4 *>(from + (min(row + u * STEP, (unsigned)N - 1) * (stride * (unsigned)sizeof(T)) + ch * 16));
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
            if (row + u * STEP < N) *(reinterpret_cast<u32x4 *>(img + (row + u * STEP) * Lds<T>::PITCH) + Lds<T>::chunk(row + u * STEP, ch)) = reg[u];
    }
};
// the zero rows behind an image's last one
template <typename T, int NA>
__device__ __forceinline__ void zero_tail(T *img, int N) {
    for (int u = N * Lds<T>::CHUNKS + threadIdx.x; u < 16 * NA * Lds<T>::CHUNKS; u += 64 * NA) {
        const u32x4 z = {0u, 0u, 0u, 0u};
        *(reinterpret_cast<u32x4 *>(img + u / Lds<T>::CHUNKS * Lds<T>::PITCH) + u % Lds<T>::CHUNKS) = z;
    }
}

template <typename T>
__device__ __forceinline__ void store4(T *p, float x, float y, float z, float w) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(x, y, z, w);
    } else {
        const f32x2 a = {x, y}, b = {z, w};
        *reinterpret_cast<uint2 *>(p) =
            make_uint2(__builtin_bit_cast(unsigned, __builtin_convertvector(a, bf16x2)), __builtin_bit_cast(unsigned, __builtin_convertvector(b, bf16x2)));
    }
}
// two accumulator tiles whose rows are d and whose column is the lane's token
template <typename T>
__device__ __forceinline__ void store_tile(T *__restrict__ base, unsigned stride, int p, int N, int lane, const f32x4 (&o)[2], float mul) {
    if (p >= N) return;
    T *dst = reinterpret_cast<T *>(reinterpret_cast<char *>(base) + ((unsigned)p * stride + 4 * (lane >> 4)) * (unsigned)sizeof(T));
#pragma unroll
    for (int h = 0; h < 2; ++h) store4(dst + 16 * h, o[h][0] * mul, o[h][1] * mul, o[h][2] * mul, o[h][3] * mul);
}

// ---- the softmax of one query tile ---------------------------------------------------------------------------------------------------------------
// over the four lanes that hold a query's keys
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float row_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}
// what is added to the wave's scores: its tiles of the bias, plus those of the mask if it says anything
template <int NA>
__device__ __forceinline__ const f32x4 *table_tiles(const float *packed, int table, int w, int lane) {
    return reinterpret_cast<const f32x4 *>(packed) + (size_t)table * (NA * NA * 64) + w * NA * 64 + lane;
}
template <int NA>
__device__ __forceinline__ void load_bias(f32x4 (&t)[NA], const float *__restrict__ packed, int head, int w, int lane) {
    const f32x4 *from = table_tiles<NA>(packed, head, w, lane);
#pragma unroll
    for (int a = 0; a < NA; ++a) t[a] = from[a * 64];
}
template <int NA>
__device__ __forceinline__ void add_mask(f32x4 (&t)[NA], const float *__restrict__ packed, const int *__restrict__ any, int heads, int win, int nW, int w, int lane) {
    if (nW == 0 || !any[(win % nW) * NA + w]) return;
    const f32x4 *from = table_tiles<NA>(packed, heads + win % nW, w, lane);
#pragma unroll
    for (int a = 0; a < NA; ++a) t[a] += from[a * 64];
}
// p: K Q^T on entry, e^(S - max) on return, 0 in the accumulators without keys -> 1 / sum, 0 for a row that has nothing left
template <int NS, int NA = tiles_of(NS)>
__device__ __forceinline__ float softmax_tile(f32x4 (&p)[NA], const f32x4 (&added)[NA], float scale) {
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        p[s >> 2][s & 3] = fmaf(p[s >> 2][s & 3], scale, added[s >> 2][s & 3]);
        m = fmaxf(m, p[s >> 2][s & 3]);
    }
    m = row_max(m);
    if (m == -INFINITY) m = 0.f;                      // nothing left: every term is 0
#pragma unroll
    for (int s = 0; s < 4 * NA; ++s) {
        p[s >> 2][s & 3] = s < NS ? ex2((p[s >> 2][s & 3] - m) * 1.4426950408889634f) : 0.f;
        l += p[s >> 2][s & 3];
    }
    l = row_sum(l);
    return l == 0.f ? 0.f : 1.f / l;
}

// ---- tables --------------------------------------------------------------------------------------------------------------------------------------
// bias [heads][N][N], then mask [nW][N][N], into the accumulator layout [query tile][key tile][lane][e]: padded keys -inf in the bias and 0 in the mask,
// padded queries 0; any[NA m + b] = query tile b of mask m has a nonzero entry.  A workgroup per table and query tile, all of a thread's loads at once (361
// masks of 49 x 49: 8.6 us with a workgroup per table)
template <int NA>
__global__ __launch_bounds__(256) void window_tables(const float *__restrict__ bias, const float *__restrict__ mask, float *__restrict__ packed, int *__restrict__ any,
                                                     int heads, int N) {
    const int t = blockIdx.x, b = blockIdx.y, e = threadIdx.x & 3, lane = threadIdx.x >> 2, i = 16 * b + (lane & 15);
    const float *src = t < heads ? bias + (size_t)t * N * N : mask + (size_t)(t - heads) * N * N;
    const float pad = t < heads ? -INFINITY : 0.f;
    float v[NA];
#pragma unroll
    for (int a = 0; a < NA; ++a) {
        const int j = 16 * a + token_of(lane >> 4, e, spread_tile(a, (N + 3) / 4));
        v[a] = src[min(i, N - 1) * N + min(j, N - 1)];
        v[a] = j >= N ? pad : (i < N ? v[a] : 0.f);
    }
    int nonzero = 0;
#pragma unroll
    for (int a = 0; a < NA; ++a) {
        packed[((size_t)t * NA + b) * (NA * 256) + a * 256 + threadIdx.x] = v[a];
        nonzero |= v[a] != 0.f;
    }
    nonzero = __syncthreads_or(nonzero);
    if (t >= heads && threadIdx.x == 0) any[(t - heads) * NA + b] = nonzero;
}

// Workgroups that share windows -- neighbouring heads, whose rows share cache lines -- sit on one of the eight chiplets: consecutive logical ids do.
__device__ __forceinline__ int logical_block() {
    const int n = gridDim.x, id = blockIdx.x, q = n / 8, rem = n % 8, x = id % 8;
    return (x < rem ? x * (q + 1) : rem * (q + 1) + (x - rem) * q) + id / 8;
}

// waves per SIMD that the registers leave room for (7 x 7 windows, stage 1: forward fp32 5 without the bias in registers level, bf16 4 and 6 without it 24
// and 27 against 23 us; backward 4, then with P and dS crossing one after the other, level, 2: 143 against 130 us, bf16 59 against 54).  At 61 to 64 tokens the
// bf16 forward's 5 leave 17 registers in scratch (40 bytes a lane); no other bound was measured there.
template <typename T>
constexpr int kFwdWaves = sizeof(T) == 4 ? 4 : 5;
constexpr int kBwdWaves = 3;

template <typename T, int NS, int NA = tiles_of(NS)>
__global__ __launch_bounds__(64 * NA, kFwdWaves<T>) void window_train_fwd(const T *__restrict__ qkv, const float *__restrict__ packed, const int *__restrict__ any,
                                                                          T *__restrict__ out, int windows, int nslab, int nW, int heads, int N, float scale) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    constexpr size_t img = image_elems<T>(NA);
    T *Q = reinterpret_cast<T *>(lds), *K = Q + img, *V = K + img;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = 16 * w + (lane & 15);
    const int job = logical_block(), slab = job / heads, head = job - slab * heads;
    const int C = heads * D, stride = 3 * C;
    const long wstride = (long)N * stride;
    const T *base = qkv + (size_t)head * D;
    Stage<T, NA> sq, sk, sv;
    auto fetch = [&](int win) {
        const T *q = base + (size_t)win * wstride;
        sq.load(q, stride, N), sk.load(q + C, stride, N), sv.load(q + 2 * C, stride, N);
    };
    auto none = [&]() { sq.clear(), sk.clear(), sv.clear(); };          // a value on both ways: else the old one would stay live through the loop
    f32x4 bias[NA];
    load_bias<NA>(bias, packed, head, w, lane);
    fetch(slab);
    zero_tail<T, NA>(Q, N), zero_tail<T, NA>(K, N), zero_tail<T, NA>(V, N);
    for (int win = slab; win < windows; win += nslab) {
        __syncthreads();                               // the previous window's images are read
        sq.store(Q, N), sk.store(K, N), sv.store(V, N);
        f32x4 added[NA];
#pragma unroll
        for (int a = 0; a < NA; ++a) added[a] = bias[a];
        add_mask<NA>(added, packed, any, heads, win, nW, w, lane);
        win + nslab < windows ? fetch(win + nslab) : none();          // behind the mask: what is asked for first arrives first
        __syncthreads();
        f32x4 p[NA], o[2] = {kZero4, kZero4};
#pragma unroll
        for (int a = 0; a < NA; ++a) p[a] = kZero4;
        Lds<T>::template rows_product<NS>(p, K, Q, w, lane);
        const float inv = softmax_tile<NS>(p, added, scale);
        Lds<T>::template columns_product<NS>(o, V, Lds<T>::template operand<NA>(p), lane);
        store_tile(out + (size_t)win * N * C + (size_t)head * D, C, i, N, lane, o, inv);
    }
}

template <typename T, int NS, int NA = tiles_of(NS)>
__global__ __launch_bounds__(64 * NA, kBwdWaves) void window_train_bwd(const T *__restrict__ qkv, const float *__restrict__ packed, const int *__restrict__ any,
                                                                       const T *__restrict__ dout, T *__restrict__ dqkv, float *__restrict__ slabs, int windows, int nslab, int nW,
                                                                       int heads, int N, float scale) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    constexpr size_t img = image_elems<T>(NA);
    T *Q = reinterpret_cast<T *>(lds), *G = Q + img, *K = G + img, *V = K + img;
    T *X = K, *Y = X + Lds<T>::cross_bytes(NA) / sizeof(T);            // P and dS cross where K and V were
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = 16 * w + (lane & 15), j = 16 * w + token_of_row(lane & 15, spread_tile(w, NS));
    const int job = logical_block(), slab = job / heads, head = job - slab * heads;
    const int C = heads * D, stride = 3 * C;
    const long wstride = (long)N * stride;
    const T *base = qkv + (size_t)head * D, *gbase = dout + (size_t)head * D;
    Stage<T, NA> sq, sk, sv, sg;
    auto fetch = [&](int win) {
        const T *q = base + (size_t)win * wstride;
        sq.load(q, stride, N), sk.load(q + C, stride, N), sv.load(q + 2 * C, stride, N);
        sg.load(gbase + (size_t)win * N * C, C, N);
    };
    auto none = [&]() { sq.clear(), sk.clear(), sv.clear(), sg.clear(); };
    fetch(slab);
    zero_tail<T, NA>(Q, N), zero_tail<T, NA>(G, N);
    f32x4 db[NA];
#pragma unroll
    for (int a = 0; a < NA; ++a) db[a] = kZero4;
    for (int win = slab; win < windows; win += nslab) {
        __syncthreads();                               // the previous window's images are read
        sq.store(Q, N), sk.store(K, N), sv.store(V, N), sg.store(G, N);
        zero_tail<T, NA>(K, N), zero_tail<T, NA>(V, N);
        f32x4 added[NA];
        int table = head;
        asm volatile("" : "+s"(table));                // loaded anew: kept over the loop it would not fit the registers
        load_bias<NA>(added, packed, table, w, lane);
        add_mask<NA>(added, packed, any, heads, win, nW, w, lane);
        __syncthreads();
        T *dq = dqkv + (size_t)win * wstride + (size_t)head * D;
        f32x4 p[NA], ds[NA];
#pragma unroll
        for (int a = 0; a < NA; ++a) p[a] = ds[a] = kZero4;
        Lds<T>::template rows_product<NS>(p, K, Q, w, lane);
        const float inv = softmax_tile<NS>(p, added, scale);
        Lds<T>::template rows_product<NS>(ds, V, G, w, lane);
        float dot = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            p[s >> 2][s & 3] = i < N ? p[s >> 2][s & 3] * inv : 0.f;              // a query row behind the window holds nothing
            dot = fmaf(p[s >> 2][s & 3], ds[s >> 2][s & 3], dot);
        }
        dot = row_sum(dot);
#pragma unroll
        for (int s = 0; s < 4 * NA; ++s) {
            ds[s >> 2][s & 3] = s < NS ? p[s >> 2][s & 3] * (ds[s >> 2][s & 3] - dot) : 0.f;
            db[s >> 2][s & 3] += ds[s >> 2][s & 3];
        }
        const auto po = Lds<T>::template operand<NA>(p), so = Lds<T>::template operand<NA>(ds);
        {
            f32x4 o[2] = {kZero4, kZero4};
            Lds<T>::template columns_product<NS>(o, K, so, lane);
            store_tile(dq, stride, i, N, lane, o, scale);
        }
        __syncthreads();                               // K and V are read
        Lds<T>::template cross_write<NA>(X, po, w, lane);
        Lds<T>::template cross_write<NA>(Y, so, w, lane);
        __syncthreads();                               // every query row of P and dS is there
        win + nslab < windows ? fetch(win + nslab) : none();          // (not before: the registers are the scores' until here)
        {
            f32x4 o[2] = {kZero4, kZero4};
            Lds<T>::template cross_product<NS>(o, G, X, w, lane);
            store_tile(dq + 2 * C, stride, j, N, lane, o, 1.f);
        }
        {
            f32x4 o[2] = {kZero4, kZero4};
            Lds<T>::template cross_product<NS>(o, Q, Y, w, lane);
            store_tile(dq + C, stride, j, N, lane, o, scale);
        }
    }
    f32x4 *to = reinterpret_cast<f32x4 *>(slabs + (size_t)job * (NA * NA * 256)) + w * NA * 64 + lane;
#pragma unroll
    for (int a = 0; a < NA; ++a) to[a * 64] = db[a];
}

// dbias[head][i][j] = the sum of the slabs, unpacked.  Sixteen waves take every sixteenth slab of the same 64 float4 each; their sums join in wave order.
template <int NA>
__global__ __launch_bounds__(1024) void window_train_dbias(const float *__restrict__ slabs, float *__restrict__ dbias, int nslab, int heads, int N) {
    __shared__ float4 part[16][64];
    const int head = blockIdx.y, lane = threadIdx.x & 63, wv = threadIdx.x >> 6, ab = blockIdx.x;      // one pair of tiles
    const float4 *src = reinterpret_cast<const float4 *>(slabs) + ((size_t)head * (NA * NA) + ab) * 64 + lane;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = wv; k < nslab; k += 16) {
        const float4 v = src[(size_t)k * heads * (NA * NA * 64)];
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
    const bool spread = spread_tile(ab % NA, (N + 3) / 4);
    const int j = 16 * (ab % NA) + token_of(lane >> 4, 0, spread), step = spread ? 4 : 1, i = 16 * (ab / NA) + (lane & 15);
    if (i >= N) return;
    float *to = dbias + ((size_t)head * N + i) * N + j;
    if (j < N) to[0] = s.x;
    if (j + step < N) to[step] = s.y;
    if (j + 2 * step < N) to[2 * step] = s.z;
    if (j + 3 * step < N) to[3 * step] = s.w;
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------------------
// Workgroups of a pass: as many as fit the 256 CUs at once (`per_cu`, by LDS and registers), each with the same number of windows but for the last ones.
int slabs_for(long windows, int heads, int per_cu) {
    const long per = (windows * heads + 256L * per_cu - 1) / (256L * per_cu);
    return (int)((windows + per - 1) / per);
}
constexpr int steps(int N) { return (N + 3) / 4; }
constexpr int tiles(int N) { return tiles_of(steps(N)); }
template <typename T>
size_t fwd_lds(int NA) { return 3 * image_elems<T>(NA) * sizeof(T); }
template <typename T>
size_t bwd_lds(int NA) {
    const size_t two = 2 * image_elems<T>(NA) * sizeof(T), cross = 2 * Lds<T>::cross_bytes(NA);
    return two + (two > cross ? two : cross);
}
int per_cu(size_t lds, int waves_per_simd, int NA) {
    const int by_lds = (int)(160 * 1024 / (lds + 512)), by_waves = 4 * waves_per_simd / NA;
    return by_lds < by_waves ? by_lds : by_waves;
}
template <typename T>
int bwd_slabs(long windows, int heads, int N) { return slabs_for(windows, heads, per_cu(bwd_lds<T>(tiles(N)), kBwdWaves, tiles(N))); }

constexpr int kMaxTables = 0xffffff;                                  // a workgroup of 256 threads each: a launch holds fewer than 2^32 threads
bool shape_ok(long windows, int heads, int N) { return windows > 0 && heads > 0 && heads <= 65535 && windows <= 0x3fffffffL / heads && N >= 1 && N <= 64; }
size_t table_elems(int N) { return (size_t)tiles(N) * tiles(N) * 256; }
size_t table_floats(int heads, int nW, int N) { return (size_t)(heads + nW) * table_elems(N); }

int check_args(const void *qkv, const float *packed, size_t packed_floats, int dtype, long windows, int nW, int heads, int N, int d) {
    if (!qkv || !packed) return SD_E_NULL;
    if (dtype != SD_F32 && dtype != SD_BF16) return SD_E_DTYPE;
    if (!sd_window_attn_train_supported(N, d)) return SD_E_UNSUPPORTED;
    if (!shape_ok(windows, heads, N) || nW < 0 || (nW > 0 && windows % nW != 0) || nW > kMaxTables - heads) return SD_E_SHAPE;
    if (packed_floats < sd_window_attn_train_packed_floats(heads, nW, N)) return SD_E_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(packed)) & 15) return SD_E_ALIGN;
    return SD_OK;
}

template <typename T, int NS, int NA = tiles_of(NS)>
int fwd_launch(const void *qkv, const float *bias, const float *mask, float *packed, void *out, long windows, int nW, int heads, int N, float scale, hipStream_t st) {
    int *any = reinterpret_cast<int *>(packed + table_floats(heads, nW, N));
    hipLaunchKernelGGL((window_tables<NA>), dim3((unsigned)(heads + nW), NA), dim3(256), 0, st, bias, mask, packed, any, heads, N);
    const size_t lds = fwd_lds<T>(NA);
    const int ns = slabs_for(windows, heads, per_cu(lds, kFwdWaves<T>, NA));
    hipLaunchKernelGGL((window_train_fwd<T, NS>), dim3((unsigned)(ns * heads)), dim3(64 * NA), lds, st, static_cast<const T *>(qkv), packed, any, static_cast<T *>(out),
                       (int)windows, ns, nW, heads, N, scale);
    return (int)hipGetLastError();
}
template <typename T, int NS, int NA = tiles_of(NS)>
int bwd_launch(const void *qkv, const float *packed, const void *dout, void *dqkv, float *dbias, long windows, int nW, int heads, int N, float scale, float *slabs,
               hipStream_t st) {
    const int *any = reinterpret_cast<const int *>(packed + table_floats(heads, nW, N));
    const int ns = bwd_slabs<T>(windows, heads, N);
    hipLaunchKernelGGL((window_train_bwd<T, NS>), dim3((unsigned)(ns * heads)), dim3(64 * NA), bwd_lds<T>(NA), st, static_cast<const T *>(qkv), packed, any,
                       static_cast<const T *>(dout), static_cast<T *>(dqkv), slabs, (int)windows, ns, nW, heads, N, scale);
    hipLaunchKernelGGL((window_train_dbias<NA>), dim3(NA * NA, (unsigned)heads), dim3(1024), 0, st, slabs, dbias, ns, heads, N);
    return (int)hipGetLastError();
}

// fn(NS as a compile-time constant) for the window's NS
template <int NS = 16, typename F>
int with_steps(int ns, F fn) {
    if constexpr (NS > 1) {
        if (ns < NS) return with_steps<NS - 1>(ns, fn);
    }
    return fn(std::integral_constant<int, NS>());
}

}  // namespace
}  // namespace sd

extern "C" {

int sd_window_attn_train_supported(int tokens_per_window, int head_dim) { return tokens_per_window >= 1 && tokens_per_window <= 64 && head_dim == sd::D; }

size_t sd_window_attn_train_packed_floats(int heads, int mask_windows, int tokens_per_window) {
    if (heads <= 0 || mask_windows < 0 || tokens_per_window < 1 || tokens_per_window > 64) return 0;
    return sd::table_floats(heads, mask_windows, tokens_per_window) + (size_t)mask_windows * sd::tiles(tokens_per_window);
}

int sd_window_attn_train_fwd(const void *qkv, const float *bias, const float *mask, float *packed, size_t packed_floats, void *out, int dtype, long windows,
                             int mask_windows, int heads, int tokens_per_window, int head_dim, float scale, void *stream) {
    const int rc = sd::check_args(qkv, packed, packed_floats, dtype, windows, mask_windows, heads, tokens_per_window, head_dim);
    if (rc != SD_OK) return rc;
    if (!out || !bias || (mask_windows > 0 && !mask)) return SD_E_NULL;
    if ((reinterpret_cast<uintptr_t>(out) & 15) || ((reinterpret_cast<uintptr_t>(bias) | reinterpret_cast<uintptr_t>(mask)) & 3)) return SD_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int N = tokens_per_window;
    return sd::with_steps(sd::steps(N), [&](auto ns) {
        return dtype == SD_F32 ? sd::fwd_launch<float, ns()>(qkv, bias, mask, packed, out, windows, mask_windows, heads, N, scale, st)
                               : sd::fwd_launch<sd::bf16_t, ns()>(qkv, bias, mask, packed, out, windows, mask_windows, heads, N, scale, st);
    });
}

size_t sd_window_attn_train_workspace_bytes(int dtype, long windows, int heads, int tokens_per_window) {
    if (!sd::shape_ok(windows, heads, tokens_per_window) || (dtype != SD_F32 && dtype != SD_BF16)) return 0;
    const int N = tokens_per_window, ns = dtype == SD_F32 ? sd::bwd_slabs<float>(windows, heads, N) : sd::bwd_slabs<sd::bf16_t>(windows, heads, N);
    return (size_t)ns * heads * sd::table_elems(N) * sizeof(float);
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
    return sd::with_steps(sd::steps(N), [&](auto ns) {
        return dtype == SD_F32 ? sd::bwd_launch<float, ns()>(qkv, packed, dout, dqkv, dbias, windows, mask_windows, heads, N, scale, slabs, st)
                               : sd::bwd_launch<sd::bf16_t, ns()>(qkv, packed, dout, dqkv, dbias, windows, mask_windows, heads, N, scale, slabs, st);
    });
}

}  // extern "C"
