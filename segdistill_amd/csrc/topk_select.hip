// topk_select.hip -- the k largest logits of every row, their indices, and what the others weigh, gfx950.
//
//   values, index : descending, equal values by ascending index (NaN counts as the largest value, -0 equals +0)
//   rest          : tau * log sum_{c not chosen} exp(x_c / tau)   (-inf when nothing is left over)
// so that softmax([values, rest] / tau) is the row's softmax with everything unchosen folded into one more class.
//
// A row is a pixel's classes (stride P: class planes [B, C, P]) or contiguous (P == 1).  Both forms read the logits once from memory and write
// k entries; the sums of the rest are taken over the unchosen terms only -- total minus chosen would cancel exactly where a confident teacher
// needs the digits -- and relative to the largest of them, so they neither overflow nor vanish.
#include <hip/hip_runtime.h>
#include <math.h>

#include "topk_device.h"

namespace sd {
namespace {

// Order-preserving integer of a value: NaN above everything, -0 == +0.  kNoKey is below every value's key.
constexpr int kNoKey = (int)0x80000000u, kMinusInfKey = (int)0x807fffffu;
__device__ __forceinline__ int key_of(float x) {
    const int b = __float_as_int(x);
    const int k = b ^ ((b >> 31) & 0x7fffffff);
    return x != x ? 0x7fffffff : (x == 0.f ? 0 : k);
}
__device__ __forceinline__ float of_key(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// ---- class planes -----------------------------------------------------------------------------------------------------------------------------
// One thread per pixel: neighbouring lanes read neighbouring pixels of a class plane.  The list of the best K so far sits in registers, sorted;
// a new element moves through it as a bubble: slot j becomes the median of (x, slot j - 1, slot j), so the sequence has no branch and no
// dynamic index.  What falls out of the list feeds the rest's running sum.  k > 32: several passes of 32, each bounded by the last entry of
// the one before (rare, and the map's second read comes from cache where it fits).
template <typename T, int K>
__global__ __launch_bounds__(256) void topk_planes(const T *__restrict__ x, T *__restrict__ values, int *__restrict__ index, float *__restrict__ rest,
                                                   int C, long P, int blocks_per_image, int k, float tau, float c2) {
    constexpr int U = 8;
    const long b = blockIdx.x / blocks_per_image;
    const long p = (long)(blockIdx.x - b * blocks_per_image) * 256 + threadIdx.x;
    if (p >= P) return;
    const T *px = x + (size_t)b * C * P + p;
    int bound_key = 0x7fffffff, bound_idx = -1;      // entries at or before this one were taken by an earlier pass
    Online low = {-INFINITY, 0.f};
    for (int base = 0; base < k; base += K) {
        const bool last = base + K >= k;
        int key[K], idx[K];
#pragma unroll
        for (int j = 0; j < K; ++j) key[j] = kNoKey, idx[j] = 0;
        for (int c0 = 0; c0 < C; c0 += U) {
            float f[U], out[U];
#pragma unroll
            for (int u = 0; u < U; ++u) f[u] = c0 + u < C ? VecIO<T>::load1(px + (size_t)(c0 + u) * P) : 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u;
                int n = key_of(f[u]);
                if (c >= C || n > bound_key || (n == bound_key && c <= bound_idx)) n = kNoKey;
                const int gone = n < key[K - 1] ? n : key[K - 1];
                out[u] = of_key(gone < kMinusInfKey ? kMinusInfKey : gone);
                int i_here = c;
#pragma unroll
                for (int j = K - 1; j >= 0; --j) {
                    const bool here = n > key[j], above = j > 0 && n > key[j > 0 ? j - 1 : 0];
                    idx[j] = above ? idx[j > 0 ? j - 1 : 0] : (here ? i_here : idx[j]);
                    key[j] = above ? key[j > 0 ? j - 1 : 0] : (here ? n : key[j]);
                }
            }
            if (last) online_fold(low, out, c2);
        }
        const int take = last ? k - base : K;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (j < take) {
                const size_t o = ((size_t)b * k + base + j) * P + p;
                VecIO<T>::store1(values + o, of_key(key[j]));
                index[o] = idx[j];
            } else {
                const float left[1] = {of_key(key[j] < kMinusInfKey ? kMinusInfKey : key[j])};
                online_fold(low, left, c2);
            }
        }
        bound_key = key[K - 1], bound_idx = idx[K - 1];
    }
    rest[(size_t)b * P + p] = low.s > 0.f || low.s != low.s ? low.m + tau * logf(low.s) : -INFINITY;
}

// ---- contiguous rows --------------------------------------------------------------------------------------------------------------------------
// NT threads per row.  1: every thread takes the maximum of its own elements; the k-th largest of these NT maxima is a lower bound of the row's
// k-th largest value (k different elements reach it).  2: elements that reach the bound -- about k of them unless the row is adverse -- go to a
// list in LDS, the others into the rest's running sum.  3: each list entry counts the entries that come before it: its rank is its place.  A
// row with more than CAP elements at the bound (constant rows, many ties) takes the k-th key exactly, by four histograms of its bytes.
template <typename T, int NT, typename F>
__device__ __forceinline__ void scan_row(const T *__restrict__ row, int V, int tid, F f) {
    constexpr int N = VecIO<T>::N;
    const int head = row_head(row, V), nvec = (V - head) / N;
    if (tid < head) {
        const float one[1] = {VecIO<T>::load1(row + tid)};
        f(one, tid);
    }
    typedef typename VecIO<T>::raw_t raw_t;
    const raw_t *v = reinterpret_cast<const raw_t *>(row + head);
    for (int i = tid; i < nvec; i += NT) {
        const raw_t r = v[i];
        float a[N];
        if constexpr (N == 4) {
#pragma unroll
            for (int q = 0; q < 4; ++q) a[q] = r[q];
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) a[2 * q] = __uint_as_float((unsigned)r[q] << 16), a[2 * q + 1] = __uint_as_float((unsigned)r[q] & 0xffff0000u);
        }
        f(a, head + i * N);
    }
    const int t = head + nvec * N + tid;
    if (t < V) {
        const float one[1] = {VecIO<T>::load1(row + t)};
        f(one, t);
    }
}

template <int NT>
struct SelectShared {
    static constexpr int CAP = NT == 64 ? 256 : 1024;
    int max_key[NT];
    int key[CAP], idx[CAP];
    float left[CAP];
    Online tmp[NT / 64];
    int hist[256];
    int count, bound, bin, need, ties, wave_ties[NT / 64];
};

template <typename T, int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void topk_rows(const T *__restrict__ x, T *__restrict__ values, int *__restrict__ index,
                                                                 float *__restrict__ rest, long rows, int V, int k, float tau, float c2) {
    constexpr int G = NT == 64 ? 4 : 1, CAP = SelectShared<NT>::CAP;
    __shared__ SelectShared<NT> shared[G];
    SelectShared<NT> &sh = shared[NT == 64 ? threadIdx.x >> 6 : 0];
    const int tid = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
    const long r = (long)blockIdx.x * G + (NT == 64 ? threadIdx.x >> 6 : 0);
    if (r >= rows) return;                            // whole waves (NT == 64) or never (one row per workgroup)
    const T *row = x + (size_t)r * V;

    int mine = kNoKey;
    scan_row<T, NT>(row, V, tid, [&](const auto &a, int) {
        for (const float f : a) mine = max(mine, key_of(f));
    });
    sh.max_key[tid] = mine;
    if (tid == 0) sh.count = 0;
    group_sync<NT>();
    int before = 0;
    for (int u = 0; u < NT; ++u) {
        const int o = sh.max_key[u];
        before += o > mine || (o == mine && u < tid);
    }
    if (before == k - 1) sh.bound = mine;
    group_sync<NT>();
    int bound = sh.bound;

    Online low = {-INFINITY, 0.f};
    scan_row<T, NT>(row, V, tid, [&](const auto &a, int i0) {
        constexpr int N = sizeof(a) / sizeof(float);
        float out[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = key_of(a[i]);
            out[i] = a[i];
            if (n >= bound) {
                out[i] = -INFINITY;
                const int at = atomicAdd(&sh.count, 1);
                if (at < CAP) sh.key[at] = n, sh.idx[at] = i0 + i;
            }
        }
        online_fold(low, out, c2);
    });
    group_sync<NT>();
    int count = sh.count;

    if (count > CAP) {
        // the k-th key by its bytes, most significant first; `need` counts down to the number of its ties that belong to the k
        unsigned prefix = 0;
        int need = k;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int h = tid; h < 256; h += NT) sh.hist[h] = 0;
            group_sync<NT>();
            const unsigned high = shift == 24 ? 0u : ~0u << (shift + 8);
            scan_row<T, NT>(row, V, tid, [&](const auto &a, int) {
                for (const float f : a) {
                    const unsigned n = (unsigned)key_of(f) ^ 0x80000000u;
                    if ((n & high) == prefix) atomicAdd(&sh.hist[(n >> shift) & 255], 1);
                }
            });
            group_sync<NT>();
            if (tid < 64) {
                // lane l holds bins 4 l .. 4 l + 3; `above` = elements in the bins of the lanes behind it
                int h[4], sum = 0;
#pragma unroll
                for (int q = 0; q < 4; ++q) h[q] = sh.hist[4 * tid + q], sum += h[q];
                int above = 0, run = sum;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int o = __shfl_down(run, d, 64);
                    if (tid + d < 64) run += o;
                }
                above = run - sum;
#pragma unroll
                for (int q = 3; q >= 0; --q) {
                    if (above < need && above + h[q] >= need) sh.bin = 4 * tid + q, sh.need = need - above, sh.ties = h[q];
                    above += h[q];
                }
            }
            group_sync<NT>();
            prefix |= (unsigned)sh.bin << shift;
            need = sh.need;
            group_sync<NT>();
        }
        bound = (int)(prefix ^ 0x80000000u);
        const int ties = sh.ties;
        if (tid == 0) sh.count = 0;
        group_sync<NT>();
        low = {-INFINITY, 0.f};
        scan_row<T, NT>(row, V, tid, [&](const auto &a, int i0) {
            constexpr int N = sizeof(a) / sizeof(float);
            float out[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int n = key_of(a[i]);
                out[i] = n < bound ? a[i] : -INFINITY;
                if (n > bound) {
                    const int at = atomicAdd(&sh.count, 1);          // k - need of them
                    sh.key[at] = n, sh.idx[at] = i0 + i;
                }
            }
            online_fold(low, out, c2);
        });
        for (int base = 0, taken = 0; taken < need; base += NT) {    // the first `need` ties in index order; there are that many
            const int i = base + tid;
            const bool tie = i < V && key_of(VecIO<T>::load1(row + i)) == bound;
            const unsigned long long vote = __ballot(tie);
            int at = taken + __popcll(vote & ((1ull << (tid & 63)) - 1)), all = __popcll(vote);
            if constexpr (NT > 64) {
                if ((tid & 63) == 0) sh.wave_ties[tid >> 6] = all;
                __syncthreads();
                all = 0;
                for (int w = 0; w < NT / 64; ++w) {
                    if (w < (tid >> 6)) at += sh.wave_ties[w];
                    all += sh.wave_ties[w];
                }
                __syncthreads();
            }
            if (tie && at < need) sh.key[k - need + at] = bound, sh.idx[k - need + at] = i;
            taken += all;
        }
        if (tid == 0 && ties > need) {
            const Online t = {of_key(bound), (float)(ties - need)};
            low = online_merge(low, t, c2);
        }
        count = k;
        group_sync<NT>();
    }

    for (int c = tid; c < count; c += NT) {
        const int n = sh.key[c], i = sh.idx[c];
        int rank = 0;
        for (int o = 0; o < count; ++o) rank += sh.key[o] > n || (sh.key[o] == n && sh.idx[o] < i);
        if (rank < k) {
            VecIO<T>::store1(values + (size_t)r * k + rank, of_key(n));
            index[(size_t)r * k + rank] = i;
        } else {
            sh.left[rank - k] = of_key(n);           // by rank: the order of the sum does not hang on the order of arrival
        }
    }
    group_sync<NT>();
    for (int c = tid; c < count - k; c += NT) {
        const float left[1] = {sh.left[c]};
        online_fold(low, left, c2);
    }
    low = online_group<NT>(low, sh.tmp, tid, c2);
    if (tid == 0) rest[r] = low.s > 0.f || low.s != low.s ? low.m + tau * logf(low.s) : -INFINITY;
}

template <typename T>
int select_launch(const void *x, void *values, int32_t *index, float *rest, long B, int C, long P, int k, float tau, hipStream_t st) {
    const T *xi = static_cast<const T *>(x);
    T *vo = static_cast<T *>(values);
    const float c2 = kLog2e / tau;
    if (P == 1) {
        if (B > kMaxBlocks) return SD_E_SHAPE;
        if (C <= 2048 && k <= 32) {
            hipLaunchKernelGGL((topk_rows<T, 64>), dim3((unsigned)((B + 3) / 4)), dim3(256), 0, st, xi, vo, index, rest, B, C, k, tau, c2);
        } else {
            hipLaunchKernelGGL((topk_rows<T, 256>), dim3((unsigned)B), dim3(256), 0, st, xi, vo, index, rest, B, C, k, tau, c2);
        }
        return (int)hipGetLastError();
    }
    const long per = (P + 255) / 256;
    if (per > kMaxBlocks / B) return SD_E_SHAPE;
    const dim3 grid((unsigned)(per * B)), block(256);
#define SD_PLANES(K) hipLaunchKernelGGL((topk_planes<T, K>), grid, block, 0, st, xi, vo, index, rest, C, P, (int)per, k, tau, c2)
    if (k <= 4) SD_PLANES(4);
    else if (k <= 8) SD_PLANES(8);
    else if (k <= 12) SD_PLANES(12);
    else if (k <= 16) SD_PLANES(16);
    else SD_PLANES(32);
#undef SD_PLANES
    return (int)hipGetLastError();
}

}  // namespace
}  // namespace sd

extern "C" {

int sd_topk_max_entries(void) { return sd::kTopkMax; }
int sd_topk_max_classes(void) { return sd::kTopkMaxClasses; }

int sd_topk_select(const void *x, void *values, int32_t *index, float *rest, int dtype, long B, int C, long P, int k, float tau, void *stream) {
    if (!x || !values || !index || !rest) return SD_E_NULL;
    if (dtype != SD_F32 && dtype != SD_BF16) return SD_E_DTYPE;
    if (B <= 0 || C <= 0 || P <= 0 || k <= 0 || k > C || B > 0x7fffffffL || P > 0x7fffffffL || !(tau > 0.f) || !isfinite(tau)) return SD_E_SHAPE;
    if (k > sd::kTopkMax || C > sd::kTopkMaxClasses) return SD_E_UNSUPPORTED;
    const uintptr_t es = dtype == SD_F32 ? 4 : 2;
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(values)) & (es - 1)) ||
        ((reinterpret_cast<uintptr_t>(index) | reinterpret_cast<uintptr_t>(rest)) & 3))
        return SD_E_ALIGN;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return dtype == SD_F32 ? sd::select_launch<float>(x, values, index, rest, B, C, P, k, tau, st)
                           : sd::select_launch<sd::bf16_t>(x, values, index, rest, B, C, P, k, tau, st);
}

}  // extern "C"
