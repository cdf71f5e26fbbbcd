// rel_bias.hip -- a learned position bias by buckets and its gradient, gfx950.
//
//   bias[h][p] = table[index[p]][h]            p over the Nq x Nk (query, key) pairs, index[p] the pair's bucket
//   dtable[b][h] = sum_{p: index[p] = b} dbias[h][p]
//
// Both are memory bound: the H Nq Nk bias elements are written once forward and read once backward.  The gradient is a gather, not a scatter: the
// plan holds the pairs ordered by bucket (ascending within one), cut into chunks of at most 512; a wave sums a chunk, a second pass a bucket's
// chunks, both in 64 bits and in a fixed order, without atomics (in 32 bits level: 61 us both, 4.5 for one window).  The ordered list is read once for eight heads.  Buckets of single distances are diagonals of the map, a
// pair per row, and neighbouring ones lie in the same cache lines: the chunks are taken by their first pair, on one chiplet after the other, so that those
// that share lines run together (2048 x 2048 pairs, 32 buckets, 16 heads, fp32: 394 -> 318 MB fetched, 86 -> 61 us).
#include <hip/hip_runtime.h>

#include "cgd_device.h"

namespace sd {
namespace {

constexpr int kBiasHeads = 8, kChunk = 512;

template <typename T, bool VECTOR>
__global__ __launch_bounds__(256) void bucket_bias_fwd(const T *__restrict__ table, const int *__restrict__ index, T *__restrict__ out, int H, long NP) {
    constexpr int N = VECTOR ? VecIO<T>::N : 1;
    const long p = ((long)blockIdx.x * 256 + threadIdx.x) * N;
    if (p >= NP) return;
    int at[N];
#pragma unroll
    for (int i = 0; i < N; ++i) at[i] = index[p + i] * H;
    const int h0 = blockIdx.y * kBiasHeads, h1 = min(H, h0 + kBiasHeads);
    for (int h = h0; h < h1; ++h) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = VecIO<T>::load1(table + at[i] + h);
        if constexpr (VECTOR) VecIO<T>::template store<true>(out + (size_t)h * NP + p, v);
        else VecIO<T>::store1(out + (size_t)h * NP + p, v[0]);
    }
}

// one wave per (chunk, eight heads); DIRECT: chunk i is all of bucket i, the sums are the gradient itself
template <typename T, bool DIRECT>
__global__ __launch_bounds__(256) void bucket_bias_chunks(const T *__restrict__ dbias, const int *__restrict__ order, const int *__restrict__ chunk_start,
                                                          const int *__restrict__ chunk_order, float *__restrict__ part, T *__restrict__ dtable, int chunks, int H, long NP) {
    const int lane = threadIdx.x & 63;
    const int wgs = gridDim.x, id = blockIdx.x, rem = wgs % 8, xcd = id % 8;          // consecutive logical workgroups share a chiplet
    const int wg = (xcd < rem ? xcd * (wgs / 8 + 1) : rem * (wgs / 8 + 1) + (xcd - rem) * (wgs / 8)) + id / 8;
    const int nth = __builtin_amdgcn_readfirstlane(wg * 4 + (int)(threadIdx.x >> 6));
    if (nth >= chunks) return;
    const int c = chunk_order[nth];
    const int lo = chunk_start[c], hi = chunk_start[c + 1];
    const int h0 = blockIdx.y * kBiasHeads, h1 = min(H, h0 + kBiasHeads);
    auto put = [&](int h, float s) {
        if constexpr (DIRECT) VecIO<T>::store1(dtable + (size_t)c * H + h, s);
        else part[(size_t)c * H + h] = s;
    };
    if (lo == hi) {                                   // an empty bucket
        for (int h = h0 + lane; h < h1; h += 64) put(h, 0.f);
        return;
    }
    int at[kChunk / 64];
    bool in[kChunk / 64];
    const int n = hi - lo;                            // (lo + 511 may lie beyond 2^31 - 1)
#pragma unroll
    for (int u = 0; u < kChunk / 64; ++u) {
        in[u] = u * 64 + lane < n;
        at[u] = order[lo + min(u * 64 + lane, n - 1)];                // lanes behind the end load the last pair again: no branch around a load
    }
    for (int h = h0; h < h1; ++h) {
        const T *d = dbias + (size_t)h * NP;
        float v[kChunk / 64];
        double s = 0;
#pragma unroll
        for (int u = 0; u < kChunk / 64; ++u) v[u] = VecIO<T>::load1(d + at[u]);
#pragma unroll
        for (int u = 0; u < kChunk / 64; ++u) s += in[u] ? v[u] : 0.f;
#pragma unroll
        for (int d2 = 32; d2 > 0; d2 >>= 1) s += __shfl_xor(s, d2, 64);
        if (lane == 0) put(h, (float)s);
    }
}

// one wave per (bucket, head): the bucket's chunk sums, in 64 bits
template <typename T>
__global__ __launch_bounds__(64) void bucket_bias_join(const float *__restrict__ part, const int *__restrict__ bucket_chunk, T *__restrict__ dtable, int H) {
    const int b = blockIdx.x, h = blockIdx.y;
    double s = 0;
#pragma unroll 8
    for (int c = bucket_chunk[b] + threadIdx.x; c < bucket_chunk[b + 1]; c += 64) s += (double)part[(size_t)c * H + h];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, 64);
    if (threadIdx.x == 0) VecIO<T>::store1(dtable + (size_t)b * H + h, (float)s);
}

template <typename T>
int fwd_launch(const void *table, const int32_t *index, void *out, int H, long NP, hipStream_t st) {
    const T *t = static_cast<const T *>(table);
    T *o = static_cast<T *>(out);
    const unsigned gy = (unsigned)((H + kBiasHeads - 1) / kBiasHeads);
    if (NP % VecIO<T>::N == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0)
        hipLaunchKernelGGL((bucket_bias_fwd<T, true>), dim3((unsigned)((NP / VecIO<T>::N + 255) / 256), gy), dim3(256), 0, st, t, index, o, H, NP);
    else
        hipLaunchKernelGGL((bucket_bias_fwd<T, false>), dim3((unsigned)((NP + 255) / 256), gy), dim3(256), 0, st, t, index, o, H, NP);
    return (int)hipGetLastError();
}

template <typename T>
int bwd_launch(const void *dbias, const int32_t *order, const int32_t *chunk_start, const int32_t *chunk_order, const int32_t *bucket_chunk,
               void *dtable, int nb, int chunks, int H, long NP,
               float *part, hipStream_t st) {
    const T *d = static_cast<const T *>(dbias);
    T *o = static_cast<T *>(dtable);
    const dim3 grid((unsigned)((chunks + 3) / 4), (unsigned)((H + kBiasHeads - 1) / kBiasHeads));
    if (chunks == nb) {
        hipLaunchKernelGGL((bucket_bias_chunks<T, true>), grid, dim3(256), 0, st, d, order, chunk_start, chunk_order, part, o, chunks, H, NP);
    } else {
        hipLaunchKernelGGL((bucket_bias_chunks<T, false>), grid, dim3(256), 0, st, d, order, chunk_start, chunk_order, part, o, chunks, H, NP);
        hipLaunchKernelGGL((bucket_bias_join<T>), dim3((unsigned)nb, (unsigned)H), dim3(64), 0, st, part, bucket_chunk, o, H);
    }
    return (int)hipGetLastError();
}

bool sizes_ok(int nb, int H, long NP) { return nb > 0 && H > 0 && NP > 0 && NP <= 0x7fffffffL && H <= 65535 && (long)nb * H <= 0x7fffffffL; }

}  // namespace
}  // namespace sd

extern "C" {

int sd_bucket_bias_chunk(void) { return sd::kChunk; }

size_t sd_bucket_bias_workspace_bytes(int buckets, int chunks, int heads) {
    return buckets > 0 && heads > 0 && chunks > buckets ? (size_t)chunks * heads * sizeof(float) : 0;
}

int sd_bucket_bias_fwd(const void *table, const int32_t *index, void *out, int dtype, int buckets, int heads, long pairs, void *stream) {
    if (!table || !index || !out) return SD_E_NULL;
    if (dtype != SD_F32 && dtype != SD_BF16) return SD_E_DTYPE;
    if (!sd::sizes_ok(buckets, heads, pairs)) return SD_E_SHAPE;
    const uintptr_t es = dtype == SD_F32 ? 3 : 1;
    if (((reinterpret_cast<uintptr_t>(table) | reinterpret_cast<uintptr_t>(out)) & es) || (reinterpret_cast<uintptr_t>(index) & 3)) return SD_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == SD_F32 ? sd::fwd_launch<float>(table, index, out, heads, pairs, st) : sd::fwd_launch<sd::bf16_t>(table, index, out, heads, pairs, st);
}

int sd_bucket_bias_bwd(const void *dbias, const int32_t *order, const int32_t *chunk_start, const int32_t *chunk_order, const int32_t *bucket_chunk, void *dtable,
                       int dtype, int buckets, int chunks, int heads, long pairs, void *workspace, size_t workspace_bytes, void *stream) {
    if (!dbias || !order || !chunk_start || !chunk_order || !bucket_chunk || !dtable) return SD_E_NULL;
    if (dtype != SD_F32 && dtype != SD_BF16) return SD_E_DTYPE;
    if (!sd::sizes_ok(buckets, heads, pairs) || chunks < buckets || chunks > 0x3ffffff) return SD_E_SHAPE;
    const size_t need = sd_bucket_bias_workspace_bytes(buckets, chunks, heads);
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3))) return SD_E_WORKSPACE;
    const uintptr_t es = dtype == SD_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(dbias) | reinterpret_cast<uintptr_t>(dtable)) & es) return SD_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    float *part = static_cast<float *>(workspace);
    return dtype == SD_F32 ? sd::bwd_launch<float>(dbias, order, chunk_start, chunk_order, bucket_chunk, dtable, buckets, chunks, heads, pairs, part, st)
                           : sd::bwd_launch<sd::bf16_t>(dbias, order, chunk_start, chunk_order, bucket_chunk, dtable, buckets, chunks, heads, pairs, part, st);
}

}  // extern "C"
