// topk_select.hip -- the k largest logits of every row, their indices, and what the others weigh, gfx950.
//
//   values, index : descending, equal values by ascending index (NaN counts as the largest value, -0 equals +0)
//   rest          : tau * log sum_{c not chosen} exp(x_c / tau)   (-inf when nothing is left over, +inf and NaN where one of those is)
// so that softmax([values, rest] / tau) is the row's softmax with everything unchosen folded into one more class.
//
// A row is a pixel's classes (stride P: class planes [B, C, P]) or contiguous (P == 1).  Both forms read the logits once from memory and write
// k entries; the sums of the rest are taken over the unchosen terms only -- total minus chosen would cancel exactly where a confident teacher
// needs the digits -- and relative to the largest of them, so they neither overflow nor vanish.
//
// Memory bound where nothing else were: N e bytes.  Measured: [8, 150, 128, 128] fp32, k = 10: 34 us (2.3 TB/s; the rounds of the search in LDS and VALU, 41 % busy), in
// bf16 36 us.  2048 rows of 65536 bf16, k = 64: 71 to 75 us (3.7 TB/s; the read alone with the group maxima 40).  One row of 32003 fp32: 8 us, a chain of latencies.
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
// dynamic index.  For more classes than the columns below hold.  What falls out of the list feeds the rest's running sum.  k > 32: several passes of 32, each bounded by the last entry of
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
            if (last) online_fold<true>(low, out, c2);
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
                online_fold<true>(low, left, c2);
            }
        }
        bound_key = key[K - 1], bound_idx = idx[K - 1];
    }
    rest[(size_t)b * P + p] = low.s > 0.f || low.s != low.s ? low.m + tau * logf(low.s) : -INFINITY;
}

// The same with the pixels' classes parked in LDS when they fit: the register list costs K steps per class; here the maxima of groups of eight classes sit in
// registers, and each of the k rounds takes the largest of them and scans its group again -- NG + 8 steps per entry instead of K per class.  Two lanes
// share a pixel, each with half of its classes in a column of its own, and exchange their best: 64 pixels per column pair leave one wave per SIMD at 150
// classes, 32 leave two (45 -> 34 us at [8, 150, 128, 128]; four lanes per pixel: 46 us, each lane scans a group per entry; the register list 84).  A taken class is
// overwritten by kNoKey, so the sum of the rest is one more pass over the columns with its maximum known.  The scans go up and compare strictly, and the
// lower half wins a tie: the lowest class does.
template <typename T, int NG>
__global__ __launch_bounds__(64) void topk_planes_lds(const T *__restrict__ x, T *__restrict__ values, int *__restrict__ index, float *__restrict__ rest, int C,
                                                      long P, int per, long tiles, int k, float tau, float c2) {
    constexpr int CL = 8 * NG;
    __shared__ int column[64 * CL];
    // half = classes per lane; for an odd count the upper half starts with the lower one's last class, which it leaves out
    const int half = (C + 1) / 2, upper = threadIdx.x >> 5, first = upper ? C - half : 0;
    const bool doubled = upper && (C & 1);
    int *mine = column + threadIdx.x;                 // class first + c at mine[64 c]
    float f[CL];
    // the next tile's loads are on their way while this one is searched
    auto fetch = [&](long tile) {
        const long b = tile / per, p = (tile - b * per) * 32 + (threadIdx.x & 31);
        const T *px = x + (size_t)b * C * P + (size_t)first * P + min(p, P - 1);
        long step = P;
        int n = half;
        asm volatile("" : "+s"(step), "+s"(n));       // offsets kept over the loop would not fit the registers: formed anew
#pragma unroll
        for (int g = 0; g < NG; ++g)
            if (8 * g < n) {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    f[8 * g + u] = VecIO<T>::load1(px);
                    px += 8 * g + u + 1 < n ? step : 0;
                }
            }
    };
    fetch(blockIdx.x);
    for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long b = tile / per, p = (tile - b * per) * 32 + (threadIdx.x & 31);
        const bool writes = !upper && p < P;
        int top[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            top[g] = kNoKey;
            if (8 * g < half) {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    int n = key_of(f[8 * g + u]);
                    if (8 * g + u >= half || (g + u == 0 && doubled)) n = kNoKey;
                    mine[64 * (8 * g + u)] = n;
                    top[g] = max(top[g], n);
                }
            }
        }
        if (tile + gridDim.x < tiles) fetch(tile + gridDim.x);
        for (int j = 0; j < k; ++j) {
            int best = top[0], bg = 0;
#pragma unroll
            for (int g = 1; g < NG; ++g) {
                const bool gt = top[g] > best;
                best = gt ? top[g] : best;
                bg = gt ? g : bg;
            }
            int *group = mine + 512 * bg;
            int at = 8, next = kNoKey;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int n = group[64 * u];
                const bool here = n == best && at == 8;
                at = here ? u : at;
                next = here ? next : max(next, n);
            }
            const int own = first + 8 * bg + at, other = __shfl_xor(best, 32, 64), other_cls = __shfl_xor(own, 32, 64);
            const bool mine_wins = best > other || (best == other && !upper);       // k <= C: the winner is a class, never padding
            if (mine_wins) {
                group[64 * at] = kNoKey;
#pragma unroll
                for (int g = 0; g < NG; ++g) top[g] = g == bg ? next : top[g];
            }
            if (writes) {
                const size_t o = ((size_t)b * k + j) * P + p;
                VecIO<T>::store1(values + o, of_key(mine_wins ? best : other));
                index[o] = mine_wins ? own : other_cls;
            }
        }
        int m = kMinusInfKey;
#pragma unroll
        for (int g = 0; g < NG; ++g) m = max(m, top[g]);
        m = max(m, __shfl_xor(m, 32, 64));
        const float ref = finite_ref<true>(of_key(m));
        float s = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
            if (8 * g < half) {
#pragma unroll
                for (int u = 0; u < 8; ++u) s += ex2((of_key(max(mine[64 * (8 * g + u)], kMinusInfKey)) - ref) * c2);      // taken: 2^-inf
            }
        s += __shfl_xor(s, 32, 64);
        if (writes) rest[(size_t)b * P + p] = s > 0.f || s != s ? ref + tau * logf(s) : -INFINITY;
    }
}

template <typename T, int NG>
int planes_lds_launch(const T *x, T *values, int32_t *index, float *rest, long B, int C, long P, int k, float tau, float c2, hipStream_t st) {
    const long per = (P + 31) / 32, tiles = per * B;
    const int lds = 64 * 8 * NG * 4, resident = lds < 10240 ? 16 : 160 * 1024 / lds;      // waves per CU
    const dim3 grid((unsigned)(tiles < 256 * resident ? tiles : 256 * resident));
    hipLaunchKernelGGL((topk_planes_lds<T, NG>), grid, dim3(64), 0, st, x, values, index, rest, C, P, (int)per, tiles, k, tau, c2);
    return (int)hipGetLastError();
}

// ---- contiguous rows --------------------------------------------------------------------------------------------------------------------------
// NT threads per row, the row in their registers: NV 16-byte vectors each (a longer row is read twice).
// 1: group maxima -- each of up to 256 groups of threads takes the largest of its elements.  The k-th largest of these maxima bounds the row's k-th
// largest value from below (k different elements reach it); one wave finds it by bisection of the ordered keys, 20 bits of them: a lower bound stays
// one.  2: elements that reach the bound -- about k of them unless the row is adverse -- go to a list in LDS, the others into the rest's sum, taken
// relative to the bound (they lie below it).  3: each list entry counts the entries before it: its rank is its place.
// A row with more than CAP elements at the bound (constant rows, many ties) takes the k-th key exactly, by four histograms of its bytes; a rest that
// lies so far below the bound that its sum loses digits is summed again relative to its own maximum.
template <typename T, int NT, int NV>
struct Row {
    static constexpr int N = VecIO<T>::N;
    typedef typename VecIO<T>::raw_t raw_t;
    const T *row;
    int V, head, nvec, tail;

    __device__ __forceinline__ Row(const T *r, int v) : row(r), V(v) {
        head = row_head(r, v);
        nvec = (v - head) / N;
        tail = head + nvec * N;
    }
    __device__ __forceinline__ bool held() const { return nvec <= NT * NV; }
    __device__ __forceinline__ raw_t vec(int i) const { return __builtin_nontemporal_load(reinterpret_cast<const raw_t *>(row + head) + i); }
    // f(values, first index): the elements before and behind the vectors
    template <typename F>
    __device__ __forceinline__ void ends(int tid, F f) const {
        if (tid < head) {
            const float one[1] = {VecIO<T>::load1(row + tid)};
            f(one, tid);
        }
        if (tail + tid < V) {
            const float one[1] = {VecIO<T>::load1(row + tail + tid)};
            f(one, tail + tid);
        }
    }
    // ... and every element of the row that is this thread's, from memory
    template <typename F>
    __device__ __forceinline__ void stream(int tid, F f) const {
#pragma unroll 1
        for (int i = tid; i < nvec; i += NT) {
            float a[N];
            unpack_vec<T>(vec(i), a);
            f(a, head + i * N);
        }
        ends(tid, f);
    }
};

template <int NT>
struct SelectShared {
    static constexpr int CAP = NT == 64 ? 256 : 1024, GROUPS = NT < 256 ? NT : 256;
    float max_of[GROUPS];
    unsigned long long entry[CAP];                    // key above, ~index below: descending keys, ascending indices
    float left[CAP], sum[NT / 64];
    Online tmp[NT / 64];
    int hist[256];
    unsigned long long last;
    int count, odd, bin, need, ties, wave_ties[NT / 64];
    float bound;
};
__device__ __forceinline__ unsigned long long entry_of(int key, int idx) { return ((unsigned long long)((unsigned)key ^ 0x80000000u) << 32) | (unsigned)~idx; }
__device__ __forceinline__ int entry_key(unsigned long long e) { return (int)((unsigned)(e >> 32) ^ 0x80000000u); }
__device__ __forceinline__ int entry_idx(unsigned long long e) { return (int)~(unsigned)e; }

// The exact way for a row that the bound does not serve: the k-th key by its bytes, most significant first, then everything above it and the first of its
// ties.  The k entries are in sh.entry on return; the sum of the others comes back per thread.
template <typename T, int NT, int NV>
__device__ __forceinline__ Online exact_entries(const Row<T, NT, NV> &row, SelectShared<NT> &sh, int tid, int k, float c2) {
    unsigned prefix = 0;
    int need = k;                                     // counts down to the number of the k-th key's ties that belong to the k
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int h = tid; h < 256; h += NT) sh.hist[h] = 0;
        group_sync<NT>();
        const unsigned high = shift == 24 ? 0u : ~0u << (shift + 8);
        row.stream(tid, [&](const auto &a, int) {
            for (const float f : a) {
                const unsigned n = (unsigned)key_of(f) ^ 0x80000000u;
                if ((n & high) == prefix) atomicAdd(&sh.hist[(n >> shift) & 255], 1);
            }
        });
        group_sync<NT>();
        if (tid < 64) {
            // lane l holds bins 4 l .. 4 l + 3; `above` = elements in the bins of the lanes behind it
            int h[4], all = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) h[q] = sh.hist[4 * tid + q], all += h[q];
            int run = all;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_down(run, d, 64);
                if (tid + d < 64) run += o;
            }
            int above = run - all;
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
    const int kth = (int)(prefix ^ 0x80000000u), ties = sh.ties;
    if (tid == 0) sh.count = 0;
    group_sync<NT>();
    Online low = {-INFINITY, 0.f};
    row.stream(tid, [&](const auto &a, int i0) {
        constexpr int N = sizeof(a) / sizeof(float);
        float out[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int n = key_of(a[i]);
            out[i] = n < kth ? a[i] : -INFINITY;
            if (n > kth) sh.entry[atomicAdd(&sh.count, 1)] = entry_of(n, i0 + i);          // k - need of them
        }
        online_fold<true>(low, out, c2);
    });
    for (int base = 0, taken = 0; taken < need; base += NT) {        // the first `need` ties in index order; there are that many
        const int i = base + tid;
        const bool tie = i < row.V && key_of(VecIO<T>::load1(row.row + i)) == kth;
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
        if (tie && at < need) sh.entry[k - need + at] = entry_of(kth, i);
        taken += all;
    }
    if (tid == 0 && ties > need) {
        const Online t = {of_key(kth), (float)(ties - need)};
        low = online_merge<true>(low, t, c2);
    }
    group_sync<NT>();
    return low;
}

template <typename T, int NT, int NV, int WAVES>
__global__ __launch_bounds__(NT == 64 ? 256 : NT, WAVES) void topk_rows(const T *__restrict__ x, T *__restrict__ values, int *__restrict__ index,
                                                                        float *__restrict__ rest, long rows, int V, int k, float tau, float c2) {
    typedef SelectShared<NT> Shared;
    typedef Row<T, NT, NV> R;
    constexpr int G = NT == 64 ? 4 : 1, CAP = Shared::CAP, GROUPS = Shared::GROUPS, N = R::N, SUB = NT / 64;
    __shared__ Shared shared[G];
    Shared &sh = shared[NT == 64 ? threadIdx.x >> 6 : 0];
    const int tid = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
    const long r = (long)blockIdx.x * G + (NT == 64 ? threadIdx.x >> 6 : 0);
    if (r >= rows) return;                            // whole waves (NT == 64) or never (one row per workgroup)
    const R row(x + (size_t)r * V, V);
    typename R::raw_t reg[NV];
    if (row.held()) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
            if (tid + u * NT < row.nvec) reg[u] = row.vec(tid + u * NT);
    }

    // 1: group maxima and the bound.  NaN elements drop out: the bound only gets lower.
    float mine = -INFINITY;
    auto largest = [&](const auto &a, int) {
        for (const float f : a) mine = fmaxf(mine, f);
    };
    if (row.held()) {
#pragma unroll
        for (int u = 0; u < NV; ++u)
            if (tid + u * NT < row.nvec) {
                float a[N];
                unpack_vec<T>(reg[u], a);
                largest(a, 0);
            }
        row.ends(tid, largest);
    } else {
        row.stream(tid, largest);
    }
#pragma unroll
    for (int d = 1; d < NT / GROUPS; d <<= 1) mine = fmaxf(mine, __shfl_xor(mine, d, 64));
    if (tid % (NT / GROUPS) == 0) sh.max_of[tid / (NT / GROUPS)] = mine;
    if (tid == 0) sh.count = sh.odd = 0;
    group_sync<NT>();
    if (tid < 64) {
        unsigned u[GROUPS / 64];
#pragma unroll
        for (int q = 0; q < GROUPS / 64; ++q) u[q] = (unsigned)key_of(sh.max_of[64 * q + tid]) ^ 0x80000000u;
        unsigned low = 0;
        for (int bit = 31; bit >= 12; --bit) {
            const unsigned trial = low | (1u << bit);
            int n = 0;
#pragma unroll
            for (int q = 0; q < GROUPS / 64; ++q) n += __popcll(__ballot(u[q] >= trial));
            if (n >= k) low = trial;
        }
        const int key = (int)(low ^ 0x80000000u);
        if (tid == 0) sh.bound = key <= kMinusInfKey ? -INFINITY : of_key(key);
    }
    group_sync<NT>();

    // 2: list and sum.  2^{x c2 - bound c2} in one rounding.  A vector without an element at the bound goes by without a look at each; a NaN that
    // passes so shows in the sum and sends the row the exact way.  At a bound of -inf everything is listed.
    const float bound = sh.bound, shift = bound * c2;
    float sum = 0.f;
    auto take = [&](const auto &a, int i0) {
        constexpr int M = sizeof(a) / sizeof(float);
        float e[M], m = a[0];
#pragma unroll
        for (int i = 0; i < M; ++i) {
            m = fmaxf(m, a[i]);
            e[i] = ex2(fmaf(a[i], c2, -shift));
        }
        if (!(m < bound)) {
#pragma unroll
            for (int i = 0; i < M; ++i)
                if (!(a[i] < bound)) {
                    e[i] = 0.f;
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < CAP) sh.entry[at] = entry_of(key_of(a[i]), i0 + i);
                }
        }
#pragma unroll
        for (int i = 0; i < M; ++i) sum += e[i];
    };
    if (row.held()) {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int i = tid + u * NT;
            if (i < row.nvec) {
                float a[N];
                unpack_vec<T>(reg[u], a);
                take(a, row.head + i * N);
            }
        }
        row.ends(tid, take);
    } else {
        row.stream(tid, take);
    }
    // NaN, or +inf: bound * c2 is below the range (every term of the sum is at most 1 otherwise)
    if (!(sum <= FLT_MAX)) sh.odd = 1;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if ((tid & 63) == 0) sh.sum[tid >> 6] = sum;
    group_sync<NT>();
    int count = sh.count;
    const bool exact = count > CAP || sh.odd;
    if (exact) {
        const Online low = online_group<NT, true>(exact_entries(row, sh, tid, k, c2), sh.tmp, tid, c2);
        if (tid == 0) sh.tmp[0] = low;
        count = k;
        group_sync<NT>();
    }

    // 3: SUB threads count for one entry
    for (int c0 = 0; c0 < count; c0 += 64) {
        const int c = c0 + tid / SUB;
        const unsigned long long e = sh.entry[min(c, count - 1)];
        int rank = 0;
        for (int o = tid % SUB; o < count; o += SUB) rank += sh.entry[o] > e;
#pragma unroll
        for (int d = 1; d < SUB; d <<= 1) rank += __shfl_xor(rank, d, 64);
        if (c < count && tid % SUB == 0) {
            const int n = entry_key(e);
            if (rank < k) {
                VecIO<T>::store1(values + (size_t)r * k + rank, of_key(n));
                index[(size_t)r * k + rank] = entry_idx(e);
                if (rank == k - 1) sh.last = e;   // the last one that is taken
            } else {
                sh.left[rank - k] = of_key(n);   // by rank: the order of the sum does not hang on the order of arrival
            }
        }
    }
    group_sync<NT>();
    Online low;
    if (exact) {
        low = sh.tmp[0];
    } else {
        float total = 0.f;
        for (int w = 0; w < SUB; ++w) total += sh.sum[w];
        Online l = {-INFINITY, 0.f};
        for (int c = tid & 63; c < count - k; c += 64) {
            const float left[1] = {sh.left[c]};
            online_fold<true>(l, left, c2);
        }
        const Online b = {total > 0.f ? bound : -INFINITY, total};
        low = count > k ? online_merge<true>(online_group<64, true>(l, nullptr, 0, c2), b, c2) : b;
        if (low.s < 0x1p-64f && k < V) {          // what is left lies far below the bound (or is -inf): relative to its own maximum
            const unsigned long long last = sh.last;
            low = {-INFINITY, 0.f};
            row.stream(tid, [&](const auto &a, int i0) {
                constexpr int M = sizeof(a) / sizeof(float);
                float out[M];
#pragma unroll
                for (int i = 0; i < M; ++i) out[i] = entry_of(key_of(a[i]), i0 + i) < last ? a[i] : -INFINITY;
                online_fold<true>(low, out, c2);
            });
            low = online_group<NT, true>(low, sh.tmp, tid, c2);
        }
    }
    if (tid == 0) rest[r] = low.s > 0.f || low.s != low.s ? low.m + tau * logf(low.s) : -INFINITY;
}

// A launch holds fewer than 2^32 threads: more rows than that go in several.
template <typename T, int NT, int NV, int WAVES>
void rows_launch_as(const T *x, T *values, int32_t *index, float *rest, long rows, int V, int k, float tau, float c2, hipStream_t st) {
    constexpr int G = NT == 64 ? 4 : 1, threads = NT == 64 ? 256 : NT;
    const long most = kMaxBlocks * 256 / threads * G;
    for (long r = 0; r < rows; r += most) {
        const long n = rows - r < most ? rows - r : most;
        hipLaunchKernelGGL((topk_rows<T, NT, NV, WAVES>), dim3((unsigned)((n + G - 1) / G)), dim3(threads), 0, st, x + (size_t)r * V, values + (size_t)r * k,
                           index + (size_t)r * k, rest + r, n, V, k, tau, c2);
    }
}

// Threads and registers by the row's bytes: a wave per row up to 8 KB (its 64 group maxima serve k <= 32), else a workgroup whose registers hold the row.
template <typename T>
int rows_launch(const T *x, T *values, int32_t *index, float *rest, long rows, int V, int k, float tau, float c2, hipStream_t st) {
    if (rows > 0x3fffffffL) return SD_E_SHAPE;
    const long bytes = (long)V * (long)sizeof(T);
#define SD_ROWS(NT, NV, WAVES) rows_launch_as<T, NT, NV, WAVES>(x, values, index, rest, rows, V, k, tau, c2, st)
    if (k <= 32 && bytes <= 2048) SD_ROWS(64, 2, 8);
    else if (k <= 32 && bytes <= 8192) SD_ROWS(64, 8, 5);
    else if (bytes <= 16384) SD_ROWS(256, 4, 6);
    else if (bytes <= 65536) SD_ROWS(256, 16, 4);
    else if (bytes <= 131072) SD_ROWS(512, 16, 4);
    else SD_ROWS(1024, 16, 4);
#undef SD_ROWS
    return (int)hipGetLastError();
}

template <typename T>
int select_launch(const void *x, void *values, int32_t *index, float *rest, long B, int C, long P, int k, float tau, hipStream_t st) {
    const T *xi = static_cast<const T *>(x);
    T *vo = static_cast<T *>(values);
    const float c2 = kLog2e / tau;
    if (P == 1) return rows_launch<T>(xi, vo, index, rest, B, C, k, tau, c2, st);
    const long per = (P + 255) / 256;
    if (per > kMaxBlocks / B) return SD_E_SHAPE;
#define SD_COLUMNS(NG) planes_lds_launch<T, NG>(xi, vo, index, rest, B, C, P, k, tau, c2, st)
    if (C <= 16) return SD_COLUMNS(1);
    if (C <= 32) return SD_COLUMNS(2);
    if (C <= 64) return SD_COLUMNS(4);
    if (C <= 160) return SD_COLUMNS(10);
    if (C <= 256) return SD_COLUMNS(16);
#undef SD_COLUMNS
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
    if (B <= 0 || C <= 0 || P <= 0 || k <= 0 || k > C || B > 0x7fffffffL || P > 0x7fffffffL || !(tau >= sd::kTauMin && tau <= sd::kTauMax)) return SD_E_SHAPE;
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
