// Layer normalisation over the last axis, forward and backward (gfx950).
//
//   forward   mu = mean x, v = mean (x - mu)^2, r = 1 / sqrt(v + eps), xh = (x - mu) r, y = xh w + b
//   backward  u = g w:  grad_x = r (u - mean u - xh mean(u xh)),  grad_w = sum_rows g xh,  grad_b = sum_rows g
//
// Bound: memory.  A row is read once into registers; mean and variance come from there in two sums (the second over
// x - mu, where a large common offset costs no more than mu's own rounding: every x - mu is shifted by up to 2^-24 |mu| and
// the rounding of the row's sum), all of it in fp32 whatever the element type.  The backward pass
// reads x and g once and writes grad_x; the row sums of grad_w / grad_b ride along in registers of a fixed grid of
// workgroups, whose partial sums a second launch adds in a fixed order (no atomics: the same inputs give the same bits).
//
// `tpr` threads share a row (a power of two): a part of a wave for short rows, a wave up to 64 * EMAX elements, several
// waves of one workgroup (exchange through LDS) above that, to 1024 threads and 16384 elements.  Longer rows take the looping kernels,
// which read the row again instead of keeping it.
//
// Built with -ffp-contract=off: u - mean(u) must cancel exactly where a row has one element.
#include "nf_common.h"

namespace {

constexpr int EMAX = 32;                 // elements of a row that a thread keeps, in workgroups up to 256 threads
constexpr int EMAX_WIDE = 16;            // in larger ones, whose threads have at most 128 registers
constexpr int LONG_SLICES = 64;          // row slices of the long rows' weight gradient

// 16 bytes of elements at the element's own alignment (global memory takes unaligned 16-byte accesses: odd row strides
// and column slices cost no other path)
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
template <typename T> struct Chunk {
    static constexpr int V = 16 / sizeof(T);
    typedef T Elems __attribute__((ext_vector_type(V)));
};

template <typename T>
__device__ __forceinline__ u32x4 load_raw(const T* p, int left) {
    constexpr int V = Chunk<T>::V;
    if (left >= V) return *reinterpret_cast<const u32x4_at2*>(p);
    typename Chunk<T>::Elems e;
#pragma unroll
    for (int k = 0; k < V; ++k) e[k] = k < left ? p[k] : (T)0.f;
    return __builtin_bit_cast(u32x4, e);
}

template <typename T>
__device__ __forceinline__ void widen(u32x4 raw, float* v) {
    const typename Chunk<T>::Elems e = __builtin_bit_cast(typename Chunk<T>::Elems, raw);
#pragma unroll
    for (int k = 0; k < Chunk<T>::V; ++k) v[k] = (float)e[k];
}

template <typename T>
__device__ __forceinline__ void load_chunk(const T* p, int left, float* v) { widen<T>(load_raw(p, left), v); }

template <typename T>
__device__ __forceinline__ void store_chunk(T* p, int left, const float* v) {
    constexpr int V = Chunk<T>::V;
    if (left >= V) {
        typename Chunk<T>::Elems e;
#pragma unroll
        for (int k = 0; k < V; ++k) e[k] = (T)v[k];
        *reinterpret_cast<u32x4_at2*>(p) = __builtin_bit_cast(u32x4, e);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k < left) p[k] = (T)v[k];
    }
}

// a chunk's part of a vector of floats (nullptr: `other` throughout)
template <int V>
__device__ __forceinline__ void load_vector(const float* p, int col, int n, float other, float* v) {
    if (p && col + V <= n) {
#pragma unroll
        for (int k = 0; k < V; k += 4) widen<float>(load_raw(p + col + k, 4), v + k);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = p && col + k < n ? p[col + k] : other;
    }
}

template <int CTRL>
__device__ __forceinline__ float add_lane(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// sum over the lanes of a row within the wave (a part of it for tpr < 64): neighbours within 16 lanes by DPP
__device__ __forceinline__ float lane_sum(float v, int tpr) {
    if (tpr >= 2) v = add_lane<0xB1>(v);                 // lane ^ 1
    if (tpr >= 4) v = add_lane<0x4E>(v);                 // lane ^ 2
    if (tpr >= 8) v = add_lane<0x141>(v);                // the other four of eight, mirrored
    if (tpr >= 16) v = add_lane<0x140>(v);               // the other eight of sixteen
    if (tpr >= 32) v += __shfl_xor(v, 16);
    if (tpr >= 64) v += __shfl_xor(v, 32);
    return v;
}

// Sums over the `tpr` threads of a row; every one of them gets them.  Rows of several waves must be summed by all threads of
// the workgroup together, through `red`: two floats per wave, twice, taken in turn (`turn`), so that one barrier does.
struct RowSum {
    float (*red)[16][2];
    int tpr, turn;
    template <int N> __device__ __forceinline__ void sums(float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = lane_sum(v[k], tpr);
        if (tpr <= 64) return;
        const int wave = threadIdx.x >> 6, per = tpr >> 6, first = wave & ~(per - 1);
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) red[turn][wave][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = 0.f;
        for (int w = first; w < first + per; ++w)
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] += red[turn][w][k];
    }
    __device__ __forceinline__ float sum(float a) {
        float v[1] = {a};
        sums(v);
        return v[0];
    }
    __device__ __forceinline__ void sum(float& a, float& b) {
        float v[2] = {a, b};
        sums(v);
        a = v[0];
        b = v[1];
    }
};

template <typename T, int C, int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_fwd_kernel(const T* __restrict__ x, int64_t xs, const float* __restrict__ w,
                                                        const float* __restrict__ b, T* __restrict__ y, int64_t ys,
                                                        float* __restrict__ mean, float* __restrict__ rstd, int64_t rows,
                                                        int n, float eps, int tpr) {
    constexpr int V = Chunk<T>::V;
    __shared__ float red[2][16][2];
    RowSum row_sum = {red, tpr, 0};
    const int t = threadIdx.x & (tpr - 1), per = blockDim.x / tpr;
    const float nf = (float)n;
    float wv[C][V], bv[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        load_vector<V>(w, (c * tpr + t) * V, n, 1.f, wv[c]);
        load_vector<V>(b, (c * tpr + t) * V, n, 0.f, bv[c]);
    }
    // the next row is requested while this one is summed where one workgroup fills a CU; smaller ones cover each other, and
    // its registers would cost them more (131072 x 2048 bf16 at one grid: 236 us without, 278 with)
    constexpr bool AHEAD = BLOCK == 1024;
    u32x4 ahead[C];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * tpr + t) * V;
            if (row < rows && col < n) ahead[c] = load_raw(x + row * xs + col, n - col);
            else ahead[c] = u32x4{0, 0, 0, 0};
        }
    };
    // (the same trip count for every thread of the workgroup: sums of several waves have a barrier)
    const int64_t stride = (int64_t)gridDim.x * per;
    int64_t row = (int64_t)blockIdx.x * per + threadIdx.x / tpr;
    if (AHEAD) fetch(row);
    for (int64_t base = (int64_t)blockIdx.x * per; base < rows; base += stride, row += stride) {
        float v[C][V], s = 0.f;
        if (!AHEAD) fetch(row);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            widen<T>(ahead[c], v[c]);
#pragma unroll
            for (int e = 0; e < V; ++e) s += v[c][e];
        }
        if (AHEAD) fetch(row + stride);
        const float mu = row_sum.sum(s) / nf;
        float q = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * tpr + t) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float d = v[c][e] - mu;
                v[c][e] = d;
                if (col + e < n) q = __builtin_fmaf(d, d, q);
            }
        }
        const float r = 1.f / sqrtf(row_sum.sum(q) / nf + eps);
        if (row >= rows) continue;
        if (t == 0 && mean) { mean[row] = mu; rstd[row] = r; }
        T* yr = y + row * ys;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * tpr + t) * V;
            if (col < n) {
#pragma unroll
                for (int e = 0; e < V; ++e) v[c][e] = __builtin_fmaf(v[c][e] * r, wv[c][e], bv[c][e]);
                store_chunk(yr + col, n - col, v[c]);
            }
        }
    }
}

// partial: [gridDim.x][2][n] (grad_w, then grad_b), each the workgroup's rows; dynamic LDS: (rows at a time) * n
// floats where a workgroup handles several rows at a time.  RAGGED: the row ends inside a chunk.  What lies past its end is
// left out by g = 0 there - and by a condition an element, since 0 times (0 - mu) r is NaN where the latter leaves fp32.  Rows of
// whole chunks are spared it (16384 x 16384 bf16, forward + backward: 608 us, with it 635; 16384 x 12001, which needs it: 744 us).
template <typename T, int C, int BLOCK, bool RAGGED>
__global__ __launch_bounds__(BLOCK) void norm_bwd_kernel(const T* __restrict__ g, int64_t gs, const T* __restrict__ x,
                                                        int64_t xs, const float* __restrict__ mean,
                                                        const float* __restrict__ rstd, const float* __restrict__ w,
                                                        T* __restrict__ gx, int64_t gxs, float* __restrict__ partial,
                                                        int64_t rows, int n, int tpr) {
    constexpr int V = Chunk<T>::V;
    extern __shared__ float lds[];
    __shared__ float red[2][16][2];
    RowSum row_sum = {red, tpr, 0};
    const int t = threadIdx.x & (tpr - 1), per = blockDim.x / tpr;
    const float nf = (float)n;
    float wv[C][V], aw[C][V], ab[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        load_vector<V>(w, (c * tpr + t) * V, n, 1.f, wv[c]);
#pragma unroll
        for (int e = 0; e < V; ++e) aw[c][e] = ab[c][e] = 0.f;
    }
    // the next row is requested while this one is summed (131072 x 2048 bf16: 430 -> 338 us); workgroups of 1024 threads have
    // no registers for it
    constexpr bool AHEAD = BLOCK < 1024;
    u32x4 ahead_x[C], ahead_g[C];
    float mu = 0.f, r = 0.f;
    auto fetch = [&](int64_t row) {
        if (row < rows) { mu = mean[row]; r = rstd[row]; }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * tpr + t) * V;
            ahead_x[c] = ahead_g[c] = u32x4{0, 0, 0, 0};
            if (row < rows && col < n) {
                ahead_x[c] = load_raw(x + row * xs + col, n - col);
                ahead_g[c] = load_raw(g + row * gs + col, n - col);
            }
        }
    };
    const int64_t stride = (int64_t)gridDim.x * per;
    int64_t row = (int64_t)blockIdx.x * per + threadIdx.x / tpr;
    if (AHEAD) fetch(row);
    for (int64_t base = (int64_t)blockIdx.x * per; base < rows; base += stride, row += stride) {
        const bool live = row < rows;
        float xh[C][V], gv[C][V], s1 = 0.f, s2 = 0.f;
        if (!AHEAD) fetch(row);
        const float rr = r;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * tpr + t) * V;
            widen<T>(ahead_x[c], xh[c]);
            widen<T>(ahead_g[c], gv[c]);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                xh[c][e] = live && col + (RAGGED ? e : 0) < n ? (xh[c][e] - mu) * r : 0.f;
                const float u = gv[c][e] * wv[c][e];
                s1 += u;
                s2 = __builtin_fmaf(u, xh[c][e], s2);
                aw[c][e] = __builtin_fmaf(gv[c][e], xh[c][e], aw[c][e]);
                ab[c][e] += gv[c][e];
            }
        }
        if (AHEAD) fetch(row + stride);
        if (!gx) continue;
        row_sum.sum(s1, s2);
        const float m1 = s1 / nf, m2 = s2 / nf;
        if (!live) continue;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * tpr + t) * V;
            if (col < n) {
                float d[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float u = gv[c][e] * wv[c][e];
                    d[e] = rr * ((u - m1) - xh[c][e] * m2);
                }
                store_chunk(gx + row * gxs + col, n - col, d);
            }
        }
    }
    if (!partial) return;
    float* out = partial + (int64_t)blockIdx.x * 2 * n;
    if (per == 1) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * tpr + t) * V;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (col + e < n) { out[col + e] = aw[c][e]; out[n + col + e] = ab[c][e]; }
        }
        return;
    }
    for (int half = 0; half < 2; ++half) {              // (one sum at a time: the LDS stays within 32 KB)
        float* mine = lds + (threadIdx.x / tpr) * n;
        __syncthreads();
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int col = (c * tpr + t) * V;
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (col + e < n) mine[col + e] = half ? ab[c][e] : aw[c][e];
        }
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += blockDim.x) {
            float s = 0.f;
            for (int k = 0; k < per; ++k) s += lds[k * n + j];
            out[half * n + j] = s;
        }
    }
}

// grad_w = sum over the partials of their first n floats, grad_b of their second n: 32 columns x 32 slices a workgroup
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float* __restrict__ partial, int count, int n,
                                                           float* __restrict__ gw, float* __restrict__ gb) {
    __shared__ float sum[32][33];
    const int64_t col = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31), all = 2 * (int64_t)n;
    const int slice = threadIdx.x >> 5;
    float s = 0.f;
    if (col < all)
#pragma unroll 4
        for (int k = slice; k < count; k += 32) s += partial[k * all + col];
    sum[slice][threadIdx.x & 31] = s;
    __syncthreads();
    if (slice == 0 && col < all) {
        for (int k = 1; k < 32; ++k) s += sum[k][threadIdx.x & 31];
        if (col < n) { if (gw) gw[col] = s; }
        else if (gb) gb[col - n] = s;
    }
}

// rows longer than 1024 threads keep: one workgroup a row, three passes over it (the later ones mostly from cache).  Measured:
// 8192 x 20000 fp32 508 us (2.6 TB/s), with the backward pass 1279; 16384 x 20000 bf16 1331 us (1.0 TB/s) and 2798.  Bound by the
// latency of each pass's loads, of which a thread has one on its way.
template <typename T>
__global__ __launch_bounds__(1024) void norm_fwd_long_kernel(const T* __restrict__ x, int64_t xs,
                                                             const float* __restrict__ w, const float* __restrict__ b,
                                                             T* __restrict__ y, int64_t ys, float* __restrict__ mean,
                                                             float* __restrict__ rstd, int64_t rows, int n, float eps) {
    constexpr int V = Chunk<T>::V;
    __shared__ float red[2][16][2];
    RowSum row_sum = {red, 1024, 0};
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * xs;
        float v[V], s = 0.f, q = 0.f;
        for (int64_t col = threadIdx.x * V; col < n; col += 1024 * V) {
            load_chunk(xr + col, (int)(n - col), v);
#pragma unroll
            for (int e = 0; e < V; ++e) s += v[e];
        }
        const float mu = row_sum.sum(s) / (float)n;
        for (int64_t col = threadIdx.x * V; col < n; col += 1024 * V) {
            load_chunk(xr + col, (int)(n - col), v);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (col + e < n) q = __builtin_fmaf(v[e] - mu, v[e] - mu, q);
        }
        const float r = 1.f / sqrtf(row_sum.sum(q) / (float)n + eps);
        if (threadIdx.x == 0 && mean) { mean[row] = mu; rstd[row] = r; }
        for (int64_t col = threadIdx.x * V; col < n; col += 1024 * V) {
            load_chunk(xr + col, (int)(n - col), v);
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (col + e < n) v[e] = __builtin_fmaf((v[e] - mu) * r, w ? w[col + e] : 1.f, b ? b[col + e] : 0.f);
            store_chunk(y + row * ys + col, (int)(n - col), v);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(1024) void norm_bwd_long_kernel(const T* __restrict__ g, int64_t gs, const T* __restrict__ x,
                                                             int64_t xs, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, const float* __restrict__ w,
                                                             T* __restrict__ gx, int64_t gxs, int64_t rows, int n) {
    constexpr int V = Chunk<T>::V;
    __shared__ float red[2][16][2];
    RowSum row_sum = {red, 1024, 0};
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float mu = mean[row], r = rstd[row];
        float xv[V], gv[V], s1 = 0.f, s2 = 0.f;
        for (int64_t col = threadIdx.x * V; col < n; col += 1024 * V) {
            load_chunk(x + row * xs + col, (int)(n - col), xv);
            load_chunk(g + row * gs + col, (int)(n - col), gv);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float u = gv[e] * ((w && col + e < n) ? w[col + e] : 1.f);
                s1 += u;
                if (col + e < n) s2 = __builtin_fmaf(u, (xv[e] - mu) * r, s2);
            }
        }
        row_sum.sum(s1, s2);
        const float m1 = s1 / (float)n, m2 = s2 / (float)n;
        for (int64_t col = threadIdx.x * V; col < n; col += 1024 * V) {
            load_chunk(x + row * xs + col, (int)(n - col), xv);
            load_chunk(g + row * gs + col, (int)(n - col), gv);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float u = gv[e] * ((w && col + e < n) ? w[col + e] : 1.f);
                xv[e] = r * ((u - m1) - ((xv[e] - mu) * r) * m2);
            }
            store_chunk(gx + row * gxs + col, (int)(n - col), xv);
        }
    }
}

// long rows' weight gradient: a thread owns V columns and walks one slice of the rows
template <typename T>
__global__ __launch_bounds__(256) void norm_wgrad_long_kernel(const T* __restrict__ g, int64_t gs, const T* __restrict__ x,
                                                              int64_t xs, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, float* __restrict__ partial,
                                                              int64_t rows, int n) {
    constexpr int V = Chunk<T>::V;
    const int64_t col = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (col >= n) return;
    float xv[V], gv[V], aw[V], ab[V];
#pragma unroll
    for (int e = 0; e < V; ++e) aw[e] = ab[e] = 0.f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float mu = mean[row], r = rstd[row];
        load_chunk(x + row * xs + col, (int)(n - col), xv);
        load_chunk(g + row * gs + col, (int)(n - col), gv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            aw[e] = __builtin_fmaf(gv[e], (xv[e] - mu) * r, aw[e]);
            ab[e] += gv[e];
        }
    }
    float* out = partial + (int64_t)blockIdx.y * 2 * n + col;
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (col + e < n) { out[e] = aw[e]; out[(int64_t)n + e] = ab[e]; }
}

// (threads a row, chunks a thread) of the register kernels, or chunks = 0: the row is too long for them
struct Split { int tpr, chunks, block, per; };

inline Split split_of(int n, int v) {
    const int64_t need = ((int64_t)n + v - 1) / v;          // chunks of the row
    Split s = {1, 1, 256, 0};
    const int few = v == 4 ? 4 : 1;                         // 16 floats or 8 halfs a thread, more only where 256 threads are too few
    while (s.tpr < 64 && s.tpr < need) s.tpr *= 2;
    while (s.chunks < few && (int64_t)s.tpr * s.chunks < need) s.chunks *= 2;
    while (s.tpr < 256 && (int64_t)s.tpr * s.chunks < need) s.tpr *= 2;
    while (s.chunks < EMAX / v && (int64_t)s.tpr * s.chunks < need) s.chunks *= 2;
    if ((int64_t)s.tpr * s.chunks < need) {
        s.tpr = s.block = 1024;
        s.chunks = (int64_t)s.tpr * (EMAX_WIDE / v) < need ? 0 : EMAX_WIDE / v;
    }
    s.per = s.block / s.tpr;
    return s;
}

// workgroups of the backward pass
inline int64_t bwd_groups(int64_t rows, const Split& s) {
    // each leaves a partial sum of 2 N floats, so no more than fit: four a CU; one where its threads take the registers of two
    // or more (16384 x 8192 bf16 forward + backward: 278 us, with 1024 of them 323)
    const int64_t need = (rows + s.per - 1) / s.per, most = s.block == 1024 || s.chunks >= 4 ? 256 : 1024;
    return need < most ? need : most;
}

template <typename T>
int launch_fwd(const void* x, int64_t xs, const float* w, const float* b, void* y, int64_t ys, float* mean, float* rstd,
               int64_t rows, int n, float eps, hipStream_t stream) {
    const Split s = split_of(n, Chunk<T>::V);
    const T* xp = (const T*)x;
    T* yp = (T*)y;
    if (!s.chunks) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_fwd_long_kernel<T>), dim3(rows < 512 ? (int)rows : 512), dim3(1024), 0,
                           stream, xp, xs, w, b, yp, ys, mean, rstd, rows, n, eps);
        return nf_launch_status();
    }
    // The vectors are read once a workgroup.  Where a thread has one chunk that is little, and more workgroups than fit keep the
    // memory evenly busy (131072 x 2048 bf16: 207 us with 8192 of them, 276 with 2048); with more chunks four a CU
    // (131072 x 512 fp32: 98 us, with eight 107), of 1024 threads two.
    const int64_t need = (rows + s.per - 1) / s.per, most = s.block == 1024 ? 512 : s.chunks > 1 ? 1024 : 8192;
    const dim3 grid((int)(need < most ? need : most)), block(s.block);
#define NF_FWD(C, BLOCK) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_fwd_kernel<T, C, BLOCK>), grid, block, 0, stream, xp, xs, w, \
                                            b, yp, ys, mean, rstd, rows, n, eps, s.tpr)
    if (s.block == 1024) NF_FWD(EMAX_WIDE / Chunk<T>::V, 1024);
    else if (s.chunks == 1) NF_FWD(1, 256);
    else if (s.chunks == 2) NF_FWD(2, 256);
    else if (s.chunks == 4) NF_FWD(4, 256);
    else if constexpr (Chunk<T>::V == 4) NF_FWD(8, 256);
#undef NF_FWD
    return nf_launch_status();
}

template <typename T>
int launch_bwd(const void* g, int64_t gs, const void* x, int64_t xs, const float* mean, const float* rstd, const float* w,
               void* gx, int64_t gxs, float* gw, float* gb, float* partial, int64_t rows, int n, hipStream_t stream) {
    const Split s = split_of(n, Chunk<T>::V);
    const T *gp = (const T*)g, *xp = (const T*)x;
    T* gxp = (T*)gx;
    const bool sums = gw || gb;
    int count = 0;
    if (!s.chunks) {
        if (gx && rows) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_bwd_long_kernel<T>), dim3(rows < 512 ? (int)rows : 512), dim3(1024), 0,
                               stream, gp, gs, xp, xs, mean, rstd, w, gxp, gxs, rows, n);
            const int e = nf_launch_status();
            if (e) return e;
        }
        if (sums && rows) {
            count = rows < LONG_SLICES ? (int)rows : LONG_SLICES;
            hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_wgrad_long_kernel<T>), dim3(nf_ceil_div(n, 256 * Chunk<T>::V), count),
                               dim3(256), 0, stream, gp, gs, xp, xs, mean, rstd, partial, rows, n);
        }
    } else if (rows) {
        count = (int)bwd_groups(rows, s);
        const dim3 grid(count), block(s.block);
        const size_t lds = (sums && s.per > 1) ? (size_t)s.per * n * sizeof(float) : 0;
        float* to = sums ? partial : nullptr;
        const bool ragged = n % Chunk<T>::V != 0;
#define NF_GO(C, BLOCK, RAGGED) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_bwd_kernel<T, C, BLOCK, RAGGED>), grid, block, lds, stream, \
                                                   gp, gs, xp, xs, mean, rstd, w, gxp, gxs, to, rows, n, s.tpr)
#define NF_BWD(C, BLOCK) do { if (ragged) NF_GO(C, BLOCK, true); else NF_GO(C, BLOCK, false); } while (0)
        if (s.block == 1024) NF_BWD(EMAX_WIDE / Chunk<T>::V, 1024);
        else if (s.chunks == 1) NF_BWD(1, 256);
        else if (s.chunks == 2) NF_BWD(2, 256);
        else if (s.chunks == 4) NF_BWD(4, 256);
        else if constexpr (Chunk<T>::V == 4) NF_BWD(8, 256);
#undef NF_BWD
#undef NF_GO
    }
    int e = nf_launch_status();
    if (e || !sums) return e;
    hipLaunchKernelGGL(norm_reduce_kernel, dim3(nf_ceil_div(2 * (int64_t)n, 32)), dim3(1024), 0, stream, partial, count, n,
                       gw, gb);
    return nf_launch_status();
}

}  // namespace

extern "C" int nf_layer_norm_fwd(const void* x, int64_t x_row_stride, const float* weight, const float* bias, void* y,
                                 int64_t y_row_stride, float* mean, float* rstd, int64_t rows, int features, double eps,
                                 int elem, void* stream) {
    const int size = nf_elem_size(elem);
    if (!size) return NF_ERR_DTYPE;
    if (rows < 0 || features < 1 || !(eps >= 0.0)) return NF_ERR_SHAPE;
    if (rows == 0) return NF_OK;
    if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return NF_ERR_NULL;
    if (x_row_stride < 0 || (rows > 1 && y_row_stride < features) || !nf_aligned(x, size) || !nf_aligned(y, size) ||
        !nf_aligned(weight, 4) || !nf_aligned(bias, 4))
        return NF_ERR_LAYOUT;
    hipStream_t s = (hipStream_t)stream;
#define NF_GO(T) launch_fwd<T>(x, x_row_stride, weight, bias, y, y_row_stride, mean, rstd, rows, features, (float)eps, s)
    return elem == NF_ELEM_F32 ? NF_GO(float) : elem == NF_ELEM_BF16 ? NF_GO(__bf16) : NF_GO(_Float16);
#undef NF_GO
}

extern "C" size_t nf_layer_norm_bwd_workspace_bytes(int64_t rows, int features, int elem) {
    const int size = nf_elem_size(elem);
    if (!size || rows < 0 || features < 1) return 0;
    const Split s = split_of(features, 16 / size);
    const int64_t count = s.chunks ? bwd_groups(rows, s) : (rows < LONG_SLICES ? rows : LONG_SLICES);
    return (size_t)count * 2 * features * sizeof(float);
}

extern "C" int nf_layer_norm_bwd(const void* grad_y, int64_t grad_y_row_stride, const void* x, int64_t x_row_stride,
                                 const float* mean, const float* rstd, const float* weight, void* grad_x,
                                 int64_t grad_x_row_stride, float* grad_weight, float* grad_bias, void* workspace,
                                 size_t workspace_bytes, int64_t rows, int features, int elem, void* stream) {
    const int size = nf_elem_size(elem);
    if (!size) return NF_ERR_DTYPE;
    if (rows < 0 || features < 1) return NF_ERR_SHAPE;
    if (!grad_x && !grad_weight && !grad_bias) return NF_OK;
    if (rows && (!grad_y || !x || !mean || !rstd)) return NF_ERR_NULL;
    if (grad_y_row_stride < 0 || x_row_stride < 0 || (grad_x && rows > 1 && grad_x_row_stride < features) ||
        !nf_aligned(grad_y, size) || !nf_aligned(x, size) || !nf_aligned(grad_x, size) || !nf_aligned(weight, 4) ||
        !nf_aligned(workspace, 4))
        return NF_ERR_LAYOUT;
    if (grad_weight || grad_bias) {
        const size_t need = nf_layer_norm_bwd_workspace_bytes(rows, features, elem);
        if (need && (!workspace || workspace_bytes < need)) return NF_ERR_SCRATCH;
    }
    hipStream_t s = (hipStream_t)stream;
#define NF_GO(T) launch_bwd<T>(grad_y, grad_y_row_stride, x, x_row_stride, mean, rstd, weight, grad_x, grad_x_row_stride,   \
                               grad_weight, grad_bias, (float*)workspace, rows, features, s)
    return elem == NF_ELEM_F32 ? NF_GO(float) : elem == NF_ELEM_BF16 ? NF_GO(__bf16) : NF_GO(_Float16);
#undef NF_GO
}
