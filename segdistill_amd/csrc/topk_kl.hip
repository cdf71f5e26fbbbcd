// topk_kl.hip -- distillation from a teacher's top logits: the criterion and its gradient, gfx950.
//
// A row holds the student's logits z_c and k entries (i_j, v_j) of the teacher, with `rest` (optional) the one logit that stands for every
// other class (topk_select.hip).  With p = softmax([v, rest] / tau), q = softmax(z / tau), A the set of the row's entry classes:
//   KL   = sum_j p_j (log p_j - log q_{i_j}) + p_r (log p_r - log q_r),     q_r = sum_{c not in A} q_c
//   dKL/dz_c * tau = q_c - sum_{j: i_j = c} p_j   (c in A),    (q_r - p_r) u_c   (c not in A),   u = softmax of z / tau over the classes not in A
// and without `rest` the same with p_r = 0 ((q_r - 0) u_c = q_c).  The streaming pass therefore takes the softmax of the classes OUTSIDE A --
// excluded one by one, not subtracted afterwards: a student that agrees with the teacher leaves q_r small -- and the entries join at the end.
//
// Each row keeps (m_r, w, m, 1/s): its gradient is w 2^{(z_c - m_r) c2} outside A, with w = (q_r - p_r) / s_r.
// Memory bound: the forward reads z, the backward reads z and writes dz; nothing of the size of z is kept between them.
// Measured: [8, 150, 128, 128] fp32, k = 10: forward 29 us (2.7 TB/s), backward 40 us (4.0 TB/s); in bf16 50 and 63 us
// (1.6 and 2.5 TB/s); 2048 rows of 65536 bf16, k = 64: forward 54 us (5.0 TB/s), backward 98 us (5.5 TB/s); the join of the row losses 2 to 5 us.
#include <hip/hip_runtime.h>
#include <math.h>

#include "topk_device.h"

namespace sd {
namespace {

struct Entries {          // one row's teacher entries lie at j * stride
    const void *values;
    const int *index;
    const float *rest;               // NULL: the entries are all the teacher says
    const unsigned char *valid;      // NULL: every row counts
    int values_bf16, k;
};
__device__ __forceinline__ float entry_value(const Entries &e, size_t at) {
    return e.values_bf16 ? VecIO<bf16_t>::load1(static_cast<const bf16_t *>(e.values) + at) : static_cast<const float *>(e.values)[at];
}

// p log(p / q) with 0 log 0 = 0, from p and the logarithm of the ratio.  A row's last steps are in 64 bits: its KL is a small difference of logarithms of
// size ten, whose rounding to 32 bits (5e-7) would be the loss's whole error where student and teacher agree.
__device__ __forceinline__ double kl_term(double p, double log_ratio) { return p > 0 || p != p ? p * log_ratio : 0.0; }

// The workgroup's sum of row losses and its number of counted rows -> part[2 * block], part[2 * block + 1].
template <int NT>
__device__ __forceinline__ void write_partial(double kl, double n, double *__restrict__ part) {
    __shared__ double acc[2 * NT / 64];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) kl += __shfl_xor(kl, d, 64), n += __shfl_xor(n, d, 64);
    if ((threadIdx.x & 63) == 0) acc[threadIdx.x >> 6] = kl, acc[NT / 64 + (threadIdx.x >> 6)] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        double a = 0, b = 0;
        for (int w = 0; w < NT / 64; ++w) a += acc[w], b += acc[NT / 64 + w];
        part[2 * (size_t)blockIdx.x] = a;
        part[2 * (size_t)blockIdx.x + 1] = b;
    }
}

__global__ __launch_bounds__(1024) void topk_kl_finish(const double *__restrict__ part, int n, float alpha, float *__restrict__ loss, float *__restrict__ inv_n) {
    double kl = 0, rows = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 1024) {
        const double2 p = reinterpret_cast<const double2 *>(part)[i];
        kl += p.x, rows += p.y;
    }
    __shared__ double acc[32];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) kl += __shfl_xor(kl, d, 64), rows += __shfl_xor(rows, d, 64);
    if ((threadIdx.x & 63) == 0) acc[threadIdx.x >> 6] = kl, acc[16 + (threadIdx.x >> 6)] = rows;
    __syncthreads();
    if (threadIdx.x == 0) {
        kl = rows = 0;
        for (int w = 0; w < 16; ++w) kl += acc[w], rows += acc[16 + w];
        const double inv = rows > 0 ? 1.0 / rows : 0.0;              // no row left: the loss and every gradient are 0
        loss[0] = (float)(kl * inv * (double)alpha);
        inv_n[0] = (float)inv;
    }
}

// ---- class planes [B, C, P]: 64 pixels per workgroup, a quarter of the classes per wave ---------------------------------------------------------
// The pixel's set A is a bit mask in LDS, a column per pixel: words[w][pixel].  Classes come by in ascending order, so the entries are met in
// ascending order too, and the rank of an entry -- the bits below it -- is its place in a second column: no search, no sort, and a class that
// appears twice has one place.  No branch per class either: a class outside A writes to (reads from) the column's spare place.
// Four waves share the pixels because one wave's walk over the classes is a chain of latencies: a map of 2 x 21 x 44 pixels and 236 classes took 50 us
// each way with one wave per 64 pixels.
constexpr int BT = 64, kWaves = 4;
struct Columns {
    unsigned *words, *ranks;
    float *vals;
    __device__ Columns(unsigned char *lds, int nwords, int lane) {
        words = reinterpret_cast<unsigned *>(lds) + lane;
        ranks = words + (size_t)nwords * BT;
        vals = reinterpret_cast<float *>(ranks + (size_t)nwords * BT);
    }
    __device__ int rank(int c) const { return (int)ranks[(c >> 5) * BT] + __popc(words[(c >> 5) * BT] & ((1u << (c & 31)) - 1)); }
};
// Eight of the pixel's entries at a time, so that their loads go out together: classes outside [0, C) become -1, their values -inf.
constexpr int kBatch = 8;
__device__ __forceinline__ void load_batch(const Entries &e, size_t at, long P, int C, int j0, int (&c)[kBatch], float (&v)[kBatch]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const size_t from = at + (size_t)min(j0 + u, e.k - 1) * P;
        c[u] = e.index[from];
        v[u] = entry_value(e, from);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
        const bool live = j0 + u < e.k && (unsigned)c[u] < (unsigned)C;
        c[u] = live ? c[u] : -1;
        v[u] = live ? v[u] : -INFINITY;
    }
}
// The mask, the ranks and the number of the classes that are listed; the teacher's maximum and normaliser over the entries and the rest.
__device__ __forceinline__ int take_entries(const Columns &col, int nwords, const Entries &e, size_t at, size_t row, long P, int C, float c2, Online &t) {
    for (int w = 0; w < nwords; ++w) col.words[w * BT] = 0;
    t = {-INFINITY, 0.f};
    for (int j0 = 0; j0 < e.k; j0 += kBatch) {
        int c[kBatch];
        float v[kBatch];
        load_batch(e, at, P, C, j0, c, v);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (c[u] >= 0) col.words[(c[u] >> 5) * BT] |= 1u << (c[u] & 31);
        online_fold(t, v, c2);
    }
    if (e.rest) {
        const float v[1] = {e.rest[row]};
        online_fold(t, v, c2);
    }
    int n = 0;
    for (int w = 0; w < nwords; ++w) col.ranks[w * BT] = n, n += __popc(col.words[w * BT]);
    return n;
}

// classes of one wave: a multiple of the eight that are fetched together
__device__ __forceinline__ int classes_per_wave(int C) { return ((C + 7) / 8 + kWaves - 1) / kWaves * 8; }

template <typename T>
__global__ __launch_bounds__(BT *kWaves) void topk_kl_planes_fwd(const T *__restrict__ S, Entries e, float4 *__restrict__ stats, double *__restrict__ part, int C, long P,
                                                                 int blocks_per_image, int nwords, float c2) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    __shared__ Online lows[kWaves][BT];
    constexpr int U = 8;                                               // divides the 32 bits of a mask word
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Columns col(lds, nwords, lane);
    const long b = blockIdx.x / blocks_per_image;
    const long p0 = (long)(blockIdx.x - b * blocks_per_image) * BT, p = p0 + lane;
    const size_t row = (size_t)b * P + p, at = (size_t)b * e.k * P + p;
    const bool active = p < P && (!e.valid || e.valid[row]);
    const int lo = min(wave * classes_per_wave(C), C), hi = min(lo + classes_per_wave(C), C);
    // the tile's address is uniform, the lane only adds its number: one scalar add per class.  A chunk is on its way while the one before it is folded.
    const T *tile = S + (size_t)b * C * P + p0;
    float z[2][U];
    auto fetch = [&](float (&to)[U], int c0) {
        const T *at_c = tile + (size_t)c0 * P;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            to[u] = c0 + u < hi ? VecIO<T>::load1(at_c + lane) : -INFINITY;
            at_c += P;
        }
    };
    Online t = {-INFINITY, 0.f}, low = {-INFINITY, 0.f};
    int members = 0;
    if (active) {
        if (lo < hi) fetch(z[0], lo);
        if (wave == 0) members = take_entries(col, nwords, e, at, row, P, C, c2, t);
    }
    __syncthreads();
    if (active && lo < hi) {
        int next = col.rank(lo);
        auto fold = [&](float (&x)[U], int c0) {
            unsigned word = col.words[(c0 >> 5) * BT] >> (c0 & 31);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool in = word & 1;
                col.vals[(in ? next : e.k) * BT] = x[u];               // place e.k is the spare one (waves share it: nobody reads it)
                next += in;
                x[u] = in ? -INFINITY : x[u];
                word >>= 1;
            }
            online_fold(low, x, c2);
        };
        for (int c0 = lo; c0 < hi; c0 += 2 * U) {
            if (c0 + U < hi) fetch(z[1], c0 + U);
            fold(z[0], c0);
            if (c0 + 2 * U < hi) fetch(z[0], c0 + 2 * U);
            if (c0 + U < hi) fold(z[1], c0 + U);
        }
    }
    lows[wave][lane] = low;
    __syncthreads();
    if (wave) return;
    double kl = 0;
    if (active) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) low = online_merge(low, lows[w][lane], c2);
        float m = low.m;
        for (int j = 0; j < members; ++j) m = fmaxf(m, col.vals[j * BT]);
        const float r = finite_ref(m);
        const float qr_num = low.s * ex2((low.m - r) * c2);
        double s = qr_num;
        for (int j = 0; j < members; ++j) s += ex2((col.vals[j * BT] - r) * c2);
        const float inv_s = (float)(1.0 / s), tr = finite_ref(t.m);
        const bool says = t.s > 0.f || t.s != t.s;
        float w = 0.f;
        if (says) {
            // the teacher's normaliser once more, then with it the terms: both walk the same entries
            const double ti = (double)c2 * (double)kLn2;
            const float er = e.rest ? ex2((e.rest[row] - tr) * c2) : 0.f;
            double ts = er, terms = 0, weights = 0;                    // sum_j e_j (v_j - z_j) / tau and sum_j e_j over the live entries
            for (int j0 = 0; j0 < e.k; j0 += kBatch) {
                int c[kBatch];
                float v[kBatch];
                load_batch(e, at, P, C, j0, c, v);
#pragma unroll
                for (int u = 0; u < kBatch; ++u)
                    if (c[u] >= 0) {
                        const float ej = ex2((v[u] - tr) * c2);
                        const double d = ((double)v[u] - (double)tr) - ((double)col.vals[col.rank(c[u]) * BT] - (double)r);
                        terms += kl_term(ej, d * ti);
                        weights += ej;
                    }
            }
            ts += weights;
            const double log_ratio = log(s) - log(ts), inv_t = 1.0 / ts;
            kl = terms * inv_t + kl_term(weights * inv_t, log_ratio);
            const double pr = er * inv_t;
            if (e.rest) kl += kl_term(pr, (((double)e.rest[row] - (double)tr) - ((double)low.m - (double)r)) * ti - log((double)low.s) + log_ratio);
            w = low.s > 0.f || low.s != low.s ? (float)((qr_num / s - pr) / low.s) : 0.f;
        }
        // a row whose teacher says nothing (no live entry, no rest) has no loss and no gradient: 1 / s = 0 and w = 0 say so to the backward
        stats[row] = says ? make_float4(finite_ref(low.m), w, r, inv_s) : make_float4(0.f, 0.f, r, 0.f);
    }
    double counted = active ? 1 : 0;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) kl += __shfl_xor(kl, d, 64), counted += __shfl_xor(counted, d, 64);
    if (lane == 0) part[2 * (size_t)blockIdx.x] = kl, part[2 * (size_t)blockIdx.x + 1] = counted;
}

template <typename T>
__global__ __launch_bounds__(BT *kWaves) void topk_kl_planes_bwd(const T *__restrict__ S, Entries e, const float4 *__restrict__ stats, const float *__restrict__ inv_n,
                                                                 const float *__restrict__ upstream, T *__restrict__ dS, int C, long P, int blocks_per_image, int nwords,
                                                                 float c2, float coef) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    constexpr int U = 8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Columns col(lds, nwords, lane);
    const long b = blockIdx.x / blocks_per_image;
    const long p0 = (long)(blockIdx.x - b * blocks_per_image) * BT, p = p0 + lane;
    const size_t row = (size_t)b * P + p, at = (size_t)b * e.k * P + p;
    const float4 st = p < P && (!e.valid || e.valid[row]) ? stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    const bool active = st.y != 0.f || st.w != 0.f;                    // otherwise the row's gradient is 0 and nothing of it is read
    const int lo = min(wave * classes_per_wave(C), C), hi = min(lo + classes_per_wave(C), C);
    const T *tile = S + (size_t)b * C * P + p0;
    T *dtile = dS + (size_t)b * C * P + p0;
    float z[2][U];
    auto fetch = [&](float (&to)[U], int c0) {
        const T *at_c = tile + (size_t)c0 * P;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            to[u] = active && c0 + u < hi ? VecIO<T>::load1(at_c + lane) : 0.f;
            at_c += P;
        }
    };
    if (lo < hi) fetch(z[0], lo);
    if (wave == 0 && active) {
        Online t;
        const int members = take_entries(col, nwords, e, at, row, P, C, c2, t);
        const float tr = finite_ref(t.m), inv_t = 1.f / t.s;
        for (int j = 0; j < members; ++j) col.vals[j * BT] = 0.f;
        for (int j0 = 0; j0 < e.k; j0 += kBatch) {
            int c[kBatch];
            float v[kBatch];
            load_batch(e, at, P, C, j0, c, v);
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (c[u] >= 0) col.vals[col.rank(c[u]) * BT] += ex2((v[u] - tr) * c2) * inv_t;
        }
    }
    __syncthreads();
    if (p >= P || lo >= hi) return;
    const float g = coef * inv_n[0] * upstream[0], w = st.y * g, inv_s = st.w;
    int next = active ? col.rank(lo) : 0;
    auto write = [&](const float (&x)[U], int c0) {
        unsigned word = active ? col.words[(c0 >> 5) * BT] >> (c0 & 31) : 0u;
        T *at_c = dtile + (size_t)c0 * P;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = word & 1;
            const float v = col.vals[(in ? next : e.k) * BT];          // (outside A: whatever the spare place holds)
            const float q = ex2((x[u] - (in ? st.z : st.x)) * c2);
            const float d = in ? fmaf(q, inv_s, -v) * g : q * w;
            next += in;
            word >>= 1;
            if (c0 + u < hi) VecIO<T>::store1(at_c + lane, active ? d : 0.f);
            at_c += P;
        }
    };
    for (int c0 = lo; c0 < hi; c0 += 2 * U) {
        if (c0 + U < hi) fetch(z[1], c0 + U);
        write(z[0], c0);
        if (c0 + 2 * U < hi) fetch(z[0], c0 + 2 * U);
        if (c0 + U < hi) write(z[1], c0 + U);
    }
}

// ---- contiguous rows [B, C]: NT threads per row ----------------------------------------------------------------------------------------------------
// A is a bit mask of the row in LDS, shifted so that an aligned 16-byte vector of logits has its bits in one byte (bf16) or half a byte (fp32).
// Every wave takes the entries by itself, two per lane: their statistics need no exchange.  Short rows are bound by what a row costs a wave whatever its length --
// the reductions over 64 lanes, the 64-bit end: 1.3 ns (65536 rows of 150 fp32: 87 us, VALU 98 % busy, backward 57; as class planes the same logits take 15).
struct RowEntries {
    int c[2];
    float v[2];
    bool first[2];     // no earlier entry names the same class
    float tr, ts;      // the teacher's finite reference and normaliser
    float rest;        // -inf where the teacher has none
};
__device__ __forceinline__ RowEntries load_entries(const Entries &e, size_t row, int C, float c2) {
    RowEntries x;
    const int lane = threadIdx.x & 63;
    Online t = {-INFINITY, 0.f};
    x.rest = e.rest ? e.rest[row] : -INFINITY;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int j = lane + 64 * h;
        x.c[h] = j < e.k ? e.index[row * e.k + j] : -1;
        if ((unsigned)x.c[h] >= (unsigned)C) x.c[h] = -1;
        x.v[h] = x.c[h] >= 0 ? entry_value(e, row * e.k + j) : -INFINITY;
        x.first[h] = x.c[h] >= 0;
    }
    online_fold(t, x.v, c2);
    t = online_group<64>(t, nullptr, 0, c2);
    if (e.rest) {
        const float v[1] = {x.rest};
        online_fold(t, v, c2);
    }
    x.tr = finite_ref(t.m);
    x.ts = t.s;
    for (int j = 0; j < e.k && j < 64; ++j) {
        const int c = __builtin_amdgcn_readlane(x.c[0], j);
        if (c == x.c[0] && j < lane) x.first[0] = false;
        if (c == x.c[1]) x.first[1] = false;
    }
    for (int j = 64; j < e.k; ++j) {
        const int c = __builtin_amdgcn_readlane(x.c[1], j - 64);
        if (c == x.c[1] && j - 64 < lane) x.first[1] = false;
    }
    return x;
}

__host__ __device__ inline int row_words(int C) { return (C + 7 + 31) / 32; }      // up to 7 bits of shift in front

// ONE: the grid holds every row, no workgroup takes a second one.  Without the loop the constants of the 64-bit logarithms are not kept in registers around it:
// 64 instead of 103, twice the waves (2048 rows of 65536 bf16: 62 -> 54 us; the loop under a bound of 80 or 64 registers spills, 78 and 84 us).  Three vectors
// in flight per lane: four spill at that bound (66 us) or leave six waves (58 us), two: 58 us.
template <typename T, int NT, bool ONE>
__global__ __launch_bounds__(NT == 64 ? 256 : NT, ONE && NT == 256 ? 8 : 1) void topk_kl_rows_fwd(const T *__restrict__ S, Entries e, float4 *__restrict__ stats, double *__restrict__ part,
                                                                        long rows, int C, float c2) {
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    constexpr int G = NT == 64 ? 4 : 1, N = VecIO<T>::N, V = 3;
    __shared__ Online tmp[NT / 64 + 1];
    const int nwords = row_words(C);
    const int grp = NT == 64 ? threadIdx.x >> 6 : 0, tid = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
    unsigned *bits = reinterpret_cast<unsigned *>(lds) + (size_t)grp * nwords;
    double kl = 0, counted = 0;
    for (int w = tid; w < nwords; w += NT) bits[w] = 0;
    for (long row = (long)blockIdx.x * G + grp; row < rows; row += (long)gridDim.x * G) {
        if (e.valid && !e.valid[row]) {                               // the same answer in all threads of the group
            if constexpr (ONE) break;
            else continue;
        }
        const T *z = S + (size_t)row * C;
        const int head = row_head(z, C), shift = (8 - (head & 7)) & 7, nvec = (C - head) / N;
        const typename VecIO<T>::raw_t *vec = reinterpret_cast<const typename VecIO<T>::raw_t *>(z + head);
        typename VecIO<T>::raw_t raw[V];
        auto fetch = [&](int i) {
#pragma unroll
            for (int u = 0; u < V; ++u) raw[u] = __builtin_nontemporal_load(vec + i + u * NT);
        };
        int i = tid;
        if (i + (V - 1) * NT < nvec) fetch(i);                         // on their way while the entries are taken
        const RowEntries x = load_entries(e, row, C, c2);
        float zj[2];                                                   // the student's logits of the entries: there when the row has been read
#pragma unroll
        for (int h = 0; h < 2; ++h) zj[h] = x.c[h] >= 0 ? VecIO<T>::load1(z + x.c[h]) : -INFINITY;
        group_sync<NT>();                                              // the mask is clear
        if (tid < 64) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (x.first[h]) atomicOr(&bits[(x.c[h] + shift) >> 5], 1u << ((x.c[h] + shift) & 31));
        }
        group_sync<NT>();
        Online low = {-INFINITY, 0.f};
        auto outside = [&](int c) { return ((bits[(c + shift) >> 5] >> ((c + shift) & 31)) & 1) == 0; };
        if (tid < head && outside(tid)) {
            const float one[1] = {VecIO<T>::load1(z + tid)};
            online_fold(low, one, c2);
        }
        // the elements of one vector that are in A leave as -inf
        auto drop = [&](float *a, int i) {
            const int at = head + shift + i * N;
            const unsigned m = bits[at >> 5] >> (at & 31);
            if (m & ((1u << N) - 1)) {
#pragma unroll
                for (int q = 0; q < N; ++q)
                    if ((m >> q) & 1) a[q] = -INFINITY;
            }
        };
        while (i + (V - 1) * NT < nvec) {                              // V vectors on their way at a time
            float a[V * N];
#pragma unroll
            for (int u = 0; u < V; ++u) {
                float v[N];
                unpack_vec<T>(raw[u], v);
                drop(v, i + u * NT);
#pragma unroll
                for (int q = 0; q < N; ++q) a[u * N + q] = v[q];
            }
            i += V * NT;
            if (i + (V - 1) * NT < nvec) fetch(i);
            online_fold(low, a, c2);
        }
        for (; i < nvec; i += NT) {
            float a[N];
            VecIO<T>::load(z + head + (size_t)i * N, a);
            drop(a, i);
            online_fold(low, a, c2);
        }
        const int t = head + nvec * N + tid;
        if (t < C && outside(t)) {
            const float one[1] = {VecIO<T>::load1(z + t)};
            online_fold(low, one, c2);
        }
        low = online_group<NT>(low, tmp, tid, c2);
        if (tid < 64) {
            const float m = wave_max(fmaxf(low.m, fmaxf(zj[0], zj[1])));
            const float r = finite_ref(m), qr_num = low.s * ex2((low.m - r) * c2);
            // every lane's share of: the student's normaliser, the teacher's, sum_j e_j (v_j - z_j) / tau
            const double ti = (double)c2 * (double)kLn2;
            double s = 0, weights = 0, terms = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s += x.first[h] ? ex2((zj[h] - r) * c2) : 0.f;
                if (x.c[h] >= 0) {
                    const float ej = ex2((x.v[h] - x.tr) * c2);
                    terms += kl_term(ej, (((double)x.v[h] - (double)x.tr) - ((double)zj[h] - (double)r)) * ti);
                    weights += ej;
                }
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d, 64), weights += __shfl_xor(weights, d, 64), terms += __shfl_xor(terms, d, 64);
            s += qr_num;
            const bool says = x.ts > 0.f || x.ts != x.ts;
            const float er = e.rest ? ex2((x.rest - x.tr) * c2) : 0.f;
            const double ts = weights + er, inv_t = 1.0 / ts, pr = er * inv_t;
            // two logarithms by one instruction stream: the even lanes' is that of s / ts, the odd ones' that of s / (ts low.s)
            const double lg = log((tid & 1 ? s / (double)low.s : s) * inv_t), lg_rest = __shfl_xor(lg, 1, 64);
            double k = terms * inv_t + kl_term(weights * inv_t, lg);
            if (e.rest) k += kl_term(pr, (((double)x.rest - (double)x.tr) - ((double)low.m - (double)r)) * ti + lg_rest);
            if (tid == 0) {
                const float w = low.s > 0.f || low.s != low.s ? (float)((qr_num / s - pr) / low.s) : 0.f;
                stats[row] = says ? make_float4(finite_ref(low.m), w, r, (float)(1.0 / s)) : make_float4(0.f, 0.f, r, 0.f);
                kl += says ? k : 0.0;
                counted += 1;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)                                // every vector of this row has been read (online_group waits for all)
                if (x.first[h]) bits[(x.c[h] + shift) >> 5] = 0;
        }
        if constexpr (ONE) break;
    }
    write_partial<NT == 64 ? 256 : NT>(kl, counted, part);
}

template <typename T, int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : NT) void topk_kl_rows_bwd(const T *__restrict__ S, Entries e, const float4 *__restrict__ stats,
                                                                        const float *__restrict__ inv_n, const float *__restrict__ upstream, T *__restrict__ dS,
                                                                        long rows, int C, float c2, float coef) {
    constexpr int G = NT == 64 ? 4 : 1, N = VecIO<T>::N;
    const int grp = NT == 64 ? threadIdx.x >> 6 : 0, tid = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
    const long row = (long)blockIdx.x * G + grp;
    if (row >= rows) return;
    const T *z = S + (size_t)row * C;
    T *d = dS + (size_t)row * C;
    const int head = row_head(z, C), nvec = (C - head) / N;
    const bool aligned = row_head(d, C) == head;                       // dS starts where S does, modulo 16 bytes
    const float4 st = !e.valid || e.valid[row] ? stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    const bool none = st.y == 0.f && st.w == 0.f;
    const float g = none ? 0.f : coef * inv_n[0] * upstream[0], w = st.y * g;
    auto grad = [&](float x) { return none ? 0.f : ex2((x - st.x) * c2) * w; };
    if (tid < head) VecIO<T>::store1(d + tid, grad(none ? 0.f : VecIO<T>::load1(z + tid)));
    for (int i = tid; i < nvec; i += NT) {
        float a[N];
        if (!none) VecIO<T>::load(z + head + (size_t)i * N, a);
#pragma unroll
        for (int q = 0; q < N; ++q) a[q] = grad(a[q]);
        if (aligned) {
            VecIO<T>::template store<false>(d + head + (size_t)i * N, a);
        } else {
#pragma unroll
            for (int q = 0; q < N; ++q) VecIO<T>::store1(d + head + (size_t)i * N + q, a[q]);
        }
    }
    const int t = head + nvec * N + tid;
    if (t < C) VecIO<T>::store1(d + t, grad(none ? 0.f : VecIO<T>::load1(z + t)));
    if (none) return;                                                   // the same answer in all threads of the group
    // the entries' classes took the outside form above; they are written again once that pass is done
    group_sync<NT>();
    if (tid < 64) {
        const RowEntries x = load_entries(e, row, C, c2);
        const float inv_t = 1.f / x.ts;
        float p[2], sum[2] = {0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 2; ++h) p[h] = x.c[h] >= 0 ? ex2((x.v[h] - x.tr) * c2) * inv_t : 0.f;
        for (int j = 0; j < e.k; ++j) {
            const int c = j < 64 ? __builtin_amdgcn_readlane(x.c[0], j) : __builtin_amdgcn_readlane(x.c[1], j - 64);
            const float pj = __int_as_float(j < 64 ? __builtin_amdgcn_readlane(__float_as_int(p[0]), j) : __builtin_amdgcn_readlane(__float_as_int(p[1]), j - 64));
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (c == x.c[h]) sum[h] += pj;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (x.first[h]) VecIO<T>::store1(d + x.c[h], (ex2((VecIO<T>::load1(z + x.c[h]) - st.z) * c2) * st.w - sum[h]) * g);
    }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------------------
struct Plan {
    int fwd, bwd, blocks, nwords, lds;     // threads per row of the two passes (P == 1); the forward's workgroups
    long per;                              // workgroups that one pass over the rows needs: the forward's (P == 1), an image's (planes)
};
// false: not a shape these kernels launch
bool plan(long B, int C, long P, int k, int element_bytes, Plan *pl) {
    if (P == 1) {
        pl->nwords = row_words(C);
        // Forward: a wave per row costs least where rows are short or many (16384 rows of 2048 fp32: 41 us, by four waves 74; of 8192: 93 against 115; 2048 of
        // 8192: 19 and 21), four waves per row are faster where they are not (1024 rows of 8192: 15, one wave 17; 1024 of 32768: 27 against 40), sixteen only for
        // few and very long ones (256 rows of 83419: 23 against 30; 512: 41 against 36; 256 of 32768: 14 both).
        // Backward, one pass without a reduction: a wave per short row (16384 rows of 1025 fp32: 40 and 44 us, bf16 29 and 42; of 4096 fp32: 105 against 93),
        // sixteen for long rows that are few (512 rows of 16384 fp32: 18 against 23; 256 of 83419: 36 against 71; 1024 of 16384: 30 both) or very long (4096 of
        // 83419: 589 against 658; 2048 of 65536 bf16: 104 against 98; 4096 of 8192: 58 against 48).
        const long bytes = (long)C * element_bytes;
        pl->fwd = C <= 2048 || (bytes <= 32768 && B >= 2048) ? 64 : B <= 256 && bytes > 131072 ? 1024 : 256;
        pl->bwd = C <= 2048 ? 64 : bytes >= 16384 && (B < 1024 || bytes > 131072) ? 1024 : 256;
        const long wgs = pl->fwd == 64 ? (B + 3) / 4 : B;
        if ((pl->bwd == 64 ? wgs : B) > kMaxBlocks) return false;
        // (16384 rows of 4000 fp32: 97 us, with at most 4096 workgroups, each with a loop, 121)
        pl->blocks = (int)(wgs < 16384 ? wgs : 16384);
        pl->lds = pl->nwords * 4 * (pl->fwd == 64 ? 4 : 1);
        pl->per = wgs;
        return true;
    }
    pl->nwords = (C + 31) / 32;
    const long column = 4L * (2 * pl->nwords + k + 1);                  // bytes of LDS per pixel
    if (column * BT > 62464) return false;                              // 64 KB less what the kernels hold besides
    pl->lds = (int)column * BT;
    pl->per = (P + BT - 1) / BT;
    if (pl->per > kMaxBlocks / B) return false;
    pl->blocks = (int)(pl->per * B);
    return true;
}

template <typename T>
int fwd_launch(const void *S, const Entries &e, long B, int C, long P, const Plan &pl, float c2, float alpha, float4 *stats, float *inv_n, float *loss, double *part,
               hipStream_t st) {
    const T *s = static_cast<const T *>(S);
    const dim3 grid((unsigned)pl.blocks);
    if (P == 1) {
#define SD_ROWS(NT, ONE) hipLaunchKernelGGL((topk_kl_rows_fwd<T, NT, ONE>), grid, dim3(NT == 64 ? 256 : NT), pl.lds, st, s, e, stats, part, B, C, c2)
        const bool one = pl.blocks == pl.per;
        if (pl.fwd == 64 && one) SD_ROWS(64, true);
        else if (pl.fwd == 64) SD_ROWS(64, false);
        else if (pl.fwd == 256 && one) SD_ROWS(256, true);
        else if (pl.fwd == 256) SD_ROWS(256, false);
        else SD_ROWS(1024, true);                      // at most 256 rows
#undef SD_ROWS
    } else {
        hipLaunchKernelGGL((topk_kl_planes_fwd<T>), grid, dim3(BT * kWaves), pl.lds, st, s, e, stats, part, C, P, (int)pl.per, pl.nwords, c2);
    }
    hipLaunchKernelGGL(topk_kl_finish, dim3(1), dim3(1024), 0, st, part, pl.blocks, alpha, loss, inv_n);
    return (int)hipGetLastError();
}

template <typename T>
int bwd_launch(const void *S, const Entries &e, long B, int C, long P, const Plan &pl, float c2, float coef, const float4 *stats, const float *inv_n,
               const float *upstream, void *dS, hipStream_t st) {
    const T *s = static_cast<const T *>(S);
    T *d = static_cast<T *>(dS);
    if (P == 1) {
        const dim3 grid((unsigned)(pl.bwd == 64 ? (B + 3) / 4 : B));
        if (pl.bwd == 64) hipLaunchKernelGGL((topk_kl_rows_bwd<T, 64>), grid, dim3(256), 0, st, s, e, stats, inv_n, upstream, d, B, C, c2, coef);
        else if (pl.bwd == 256) hipLaunchKernelGGL((topk_kl_rows_bwd<T, 256>), grid, dim3(256), 0, st, s, e, stats, inv_n, upstream, d, B, C, c2, coef);
        else hipLaunchKernelGGL((topk_kl_rows_bwd<T, 1024>), grid, dim3(1024), 0, st, s, e, stats, inv_n, upstream, d, B, C, c2, coef);
    } else {
        const dim3 grid((unsigned)pl.blocks);
        hipLaunchKernelGGL((topk_kl_planes_bwd<T>), grid, dim3(BT * kWaves), pl.lds, st, s, e, stats, inv_n, upstream, d, C, P, (int)pl.per, pl.nwords, c2, coef);
    }
    return (int)hipGetLastError();
}

int check_args(const void *S, const void *values, const int32_t *index, const float *rest, int dtype, int values_dtype, long B, int C, long P, int k, float tau,
               Plan *pl) {
    if (!S || !values || !index) return SD_E_NULL;
    if ((dtype != SD_F32 && dtype != SD_BF16) || (values_dtype != SD_F32 && values_dtype != SD_BF16)) return SD_E_DTYPE;
    if (B <= 0 || C <= 0 || P <= 0 || k <= 0 || B > 0x7fffffffL || P > 0x7fffffffL || !(tau >= kTauMin && tau <= kTauMax)) return SD_E_SHAPE;
    if (k > kTopkMax || C > kTopkMaxClasses || !plan(B, C, P, k, dtype == SD_F32 ? 4 : 2, pl)) return SD_E_UNSUPPORTED;
    const uintptr_t es = dtype == SD_F32 ? 3 : 1, ev = values_dtype == SD_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(S) & es) || (reinterpret_cast<uintptr_t>(values) & ev) ||
        ((reinterpret_cast<uintptr_t>(index) | reinterpret_cast<uintptr_t>(rest)) & 3))
        return SD_E_ALIGN;
    return SD_OK;
}

}  // namespace
}  // namespace sd

extern "C" {

int sd_topk_kl_supported(long B, int C, long P, int k) {
    sd::Plan pl;
    return B > 0 && C > 0 && P > 0 && k > 0 && B <= 0x7fffffffL && P <= 0x7fffffffL && k <= sd::kTopkMax && C <= sd::kTopkMaxClasses && sd::plan(B, C, P, k, 4, &pl);
}

size_t sd_topk_kl_workspace_bytes(long B, int C, long P, int k) {
    sd::Plan f32, bf16;                    // for logits of either type
    if (!sd_topk_kl_supported(B, C, P, k) || !sd::plan(B, C, P, k, 4, &f32) || !sd::plan(B, C, P, k, 2, &bf16)) return 0;
    return 2 * sizeof(double) * (size_t)(f32.blocks > bf16.blocks ? f32.blocks : bf16.blocks);
}

int sd_topk_kl_fwd(const void *S, const void *values, const int32_t *index, const float *rest, const uint8_t *valid, int dtype, int values_dtype, long B, int C,
                   long P, int k, float tau, float alpha, float *stats, float *inv_rows, float *loss, void *workspace, size_t workspace_bytes, void *stream) {
    sd::Plan pl;
    const int rc = sd::check_args(S, values, index, rest, dtype, values_dtype, B, C, P, k, tau, &pl);
    if (rc != SD_OK) return rc;
    if (!stats || !inv_rows || !loss || !workspace) return SD_E_NULL;
    if (workspace_bytes < 2 * sizeof(double) * (size_t)pl.blocks || (reinterpret_cast<uintptr_t>(workspace) & 15)) return SD_E_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(stats) & 15) return SD_E_ALIGN;
    const sd::Entries e = {values, index, rest, valid, values_dtype == SD_BF16, k};
    hipStream_t st = static_cast<hipStream_t>(stream);
    float4 *sv = reinterpret_cast<float4 *>(stats);
    const float c2 = sd::kLog2e / tau;
    return dtype == SD_F32 ? sd::fwd_launch<float>(S, e, B, C, P, pl, c2, alpha, sv, inv_rows, loss, static_cast<double *>(workspace), st)
                           : sd::fwd_launch<sd::bf16_t>(S, e, B, C, P, pl, c2, alpha, sv, inv_rows, loss, static_cast<double *>(workspace), st);
}

int sd_topk_kl_bwd(const void *S, const void *values, const int32_t *index, const float *rest, const uint8_t *valid, int dtype, int values_dtype, long B, int C,
                   long P, int k, float tau, float alpha, const float *stats, const float *inv_rows, const float *upstream, void *dS, void *stream) {
    sd::Plan pl;
    const int rc = sd::check_args(S, values, index, rest, dtype, values_dtype, B, C, P, k, tau, &pl);
    if (rc != SD_OK) return rc;
    if (!stats || !inv_rows || !upstream || !dS) return SD_E_NULL;
    if ((reinterpret_cast<uintptr_t>(stats) & 15) || (reinterpret_cast<uintptr_t>(dS) & (dtype == SD_F32 ? 3 : 1))) return SD_E_ALIGN;
    const sd::Entries e = {values, index, rest, valid, values_dtype == SD_BF16, k};
    hipStream_t st = static_cast<hipStream_t>(stream);
    const float4 *sv = reinterpret_cast<const float4 *>(stats);
    const float c2 = sd::kLog2e / tau, coef = alpha / tau;
    return dtype == SD_F32 ? sd::bwd_launch<float>(S, e, B, C, P, pl, c2, coef, sv, inv_rows, upstream, dS, st)
                           : sd::bwd_launch<sd::bf16_t>(S, e, B, C, P, pl, c2, coef, sv, inv_rows, upstream, dS, st);
}

}  // extern "C"
