// Orthogonalisation of matrix updates by Newton-Schulz products, and the Muon step around it (gfx950).
//
//   X0 = G / (|G|_F + eps),   steps times:  S = X X^T,  X <- a X + (b S + c S S) X,   a, b, c = 3.4445, -4.7750, 2.0315
//
// on the smaller side (G is read transposed where rows > columns, so X is m x n with m <= n).  The odd quintic
// p(s) = a s + b s^3 + c s^5 acts on every singular value: it maps [0, 1.2025] into itself (its largest value there is
// 1.2024, at s = 0.5545) and lifts small values by a each step, so after five steps all but the smallest lie near 1.
//
// Bound: matrix products, 3 m^2 n + m^3 flop a step and matrix with the symmetric halves of S and S S left out.  They run
// on the fp16 matrix pipe with both operands as two fp16 terms v = hi + lo (hi = v rounded, lo = the rest rounded: 22 to
// 23 bits) and three products hi hi + hi lo + lo hi in fp32 accumulators: the error of the whole iteration is that of fp32
// products (measured beside torch's on spectra from flat to four decades), at a third of the fp16 rate instead of the
// fp32 pipe's sixteenth.  One term is not enough even for bf16 results: five steps lift its 2^-12 to 2e-3 of the result,
// more than the result's own rounding.  Because |X|, |S| and |b S + c S S| have spectral norms below 1.21, 1.45 and 2.81,
// their elements times 2^15, 2^15 and 2^14 fit fp16, and lo keeps its bits down to 2^-39: fixed scales, no searches.
// a X is added in the epilogue, where it keeps fp32 (in the product it would cost the identity part two bits).
//
// Storage: a matrix is a grid of 32 x 32 cells of 4 KB, [k block of 16][term][lane][8 halfs], where lane = row + 32 (k / 8)
// is the operand order of v_mfma_f32_32x32x16_f16: a 1 KB piece goes from memory to LDS with one instruction of a wave and
// from LDS to registers without bank conflicts.  X is kept in both orientations (S needs rows of X, the update rows of
// X^T); the padding of a matrix to whole cells is zero and stays zero.
#include "nf_common.h"

#include <math.h>

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float CA = 3.4445f, CB = -4.7750f, CC = 2.0315f;
constexpr int CELL = 4096;               // bytes of a 32 x 32 cell
constexpr int PIECE = 1024;              // of one term of one 32 x 16 block
constexpr int MAX_GROUPS = 8;            // shapes in one sequence of launches
constexpr int MAX_MATRICES = 48;         // matrices with pointers of their own (kernel arguments) in one sequence
constexpr int NORM_BLOCKS = 256;         // partial sums of a matrix's norm

// matrices of one shape
struct Group {
    int m, n;                            // m <= n
    int sm, sn;                          // cells along each
    int trans;                           // rows > columns: X = G^T
    int count, first;                    // matrices, index of the first
    int64_t x, xt[2], s, r;              // byte offsets in the workspace; matrix i of X is at x + i * sm * sn * CELL, ...
};
struct Plan {
    Group g[MAX_GROUPS];
    int first_tile[MAX_GROUPS + 1];      // tiles of the launch, group by group
    int groups;
};
struct Pointers {
    const float* grad[MAX_MATRICES];
    float* momentum[MAX_MATRICES];
    float* param[MAX_MATRICES];
};
// the matrices of nf_orthogonalize (one group), or the scalars of the Muon step
struct Ends {
    const void* in;
    void* out;
    int64_t in_matrix, in_row, out_matrix, out_row;
    float momentum, keep, lr;
    int nesterov;
};

__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// (LDS traffic of a wave with itself: in order, but only this tells the compiler that lanes talk to each other)
__device__ __forceinline__ void wave_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Workgroups go round robin to the eight XCDs, each with an L2 of its own: XCD k gets the k-th eighth of the tiles.
__device__ __forceinline__ int xcd_order(int id, int total) {
    const int q = total >> 3, rest = total & 7, xcd = id & 7;
    return xcd * q + (xcd < rest ? xcd : rest) + (id >> 3);
}

// ---- norm and momentum -------------------------------------------------------------------------------------------------
// partial[matrix][block] = sum of squares in fp64 (no overflow or underflow over the whole fp32 range, and the same bits
// every time); MUON: momentum <- mu momentum + grad on the way, the norm is that of the update
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void orth_norm_kernel(Plan plan, Pointers ptr, Ends io, double* __restrict__ partial) {
    __shared__ double red[4];
    const int mat = blockIdx.y, blocks = gridDim.x;
    int k = 0;
    while (k + 1 < plan.groups && mat >= plan.g[k + 1].first) ++k;
    const Group& g = plan.g[k];
    const int cols = g.trans ? g.m : g.n;
    const int64_t total = (int64_t)g.m * g.n;
    double sum = 0;
    if constexpr (MUON) {
        const float* gr = ptr.grad[mat];
        float* mo = ptr.momentum[mat];
        for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)blocks * 256) {
            const float gv = gr[e], mv = __builtin_fmaf(io.momentum, mo[e], gv);
            mo[e] = mv;
            const double u = io.nesterov ? __builtin_fmaf(io.momentum, mv, gv) : mv;
            sum += u * u;
        }
    } else {
        const T* in = (const T*)io.in + mat * io.in_matrix;
        const int rows = g.trans ? g.n : g.m;
        for (int64_t row = blockIdx.x; row < rows; row += blocks)
            for (int c = threadIdx.x; c < cols; c += 256) {
                const double u = (double)(float)in[row * io.in_row + c];
                sum += u * u;
            }
    }
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partial[(int64_t)mat * NORM_BLOCKS + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- cells ---------------------------------------------------------------------------------------------------------------
// one term pair of a cell's k block q, from / to memory: this lane's 8 values of row lane % 32, columns 16 q + 8 (lane / 32)
__device__ __forceinline__ void store_terms(char* cell, int q, int lane, const float* v) {
    f16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        _Float16 h, l;
        split(v[e], h, l);
        hi[e] = h;
        lo[e] = l;
    }
    *reinterpret_cast<f16x8*>(cell + q * 2 * PIECE + lane * 16) = hi;
    *reinterpret_cast<f16x8*>(cell + q * 2 * PIECE + PIECE + lane * 16) = lo;
}

__device__ __forceinline__ void load_terms(const char* cell, int q, int lane, float* v) {
    const f16x8 hi = *reinterpret_cast<const f16x8*>(cell + q * 2 * PIECE + lane * 16);
    const f16x8 lo = *reinterpret_cast<const f16x8*>(cell + q * 2 * PIECE + PIECE + lane * 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)hi[e] + (float)lo[e];
}

// a wave's 32 x 32 floats in LDS
struct Sub {
    float (*at)[33];
    __device__ __forceinline__ void rows(int q, int lane, float* v) const {
        const int r = lane & 31, c = 16 * q + 8 * (lane >> 5);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = at[r][c + e];
    }
    __device__ __forceinline__ void put_rows(int q, int lane, const float* v) const {
        const int r = lane & 31, c = 16 * q + 8 * (lane >> 5);
#pragma unroll
        for (int e = 0; e < 8; ++e) at[r][c + e] = v[e];
    }
    __device__ __forceinline__ void columns(int q, int lane, float* v) const {
        const int r = lane & 31, c = 16 * q + 8 * (lane >> 5);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = at[c + e][r];
    }
};

// X0 in both orientations: a wave a cell
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void orth_start_kernel(Plan plan, Pointers ptr, Ends io, const double* __restrict__ partial,
                                                         int blocks, double eps, char* __restrict__ ws) {
    __shared__ float lds[4][32][33];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int k = 0;
    while (k + 1 < plan.groups && (int)blockIdx.x >= plan.first_tile[k + 1]) ++k;
    const Group& g = plan.g[k];
    const int cells = g.sm * g.sn, per = (cells + 3) >> 2;
    const int in_group = blockIdx.x - plan.first_tile[k], idx = in_group / per;
    const int cell = (in_group - idx * per) * 4 + wave;
    if (cell >= cells) return;                           // (no barriers below: the waves are independent)
    const int mat = g.first + idx, ci = cell / g.sn, cj = cell - ci * g.sn;
    double sum = 0;
    for (int e = lane; e < blocks; e += 64) sum += partial[(int64_t)mat * NORM_BLOCKS + e];
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    const double scale = 32768.0 / (sqrt(sum) + eps);
    const Sub sub = {lds[wave]};
    // rows of G (cj's cells where X is its transpose)
    const int r0 = (g.trans ? cj : ci) * 32, c0 = (g.trans ? ci : cj) * 32;
    const int rows = g.trans ? g.n : g.m, cols = g.trans ? g.m : g.n;
    const T* in = MUON ? nullptr : (const T*)io.in + mat * io.in_matrix;
    const float* gr = MUON ? ptr.grad[mat] : nullptr;
    const float* mo = MUON ? ptr.momentum[mat] : nullptr;
#pragma unroll 4
    for (int it = 0; it < 16; ++it) {
        const int r = it * 2 + (lane >> 5), c = lane & 31;
        float v = 0.f;
        if (r0 + r < rows && c0 + c < cols) {
            if constexpr (MUON) {
                const int64_t e = (int64_t)(r0 + r) * cols + c0 + c;
                v = mo[e];
                if (io.nesterov) v = __builtin_fmaf(io.momentum, v, gr[e]);
            } else {
                v = (float)in[(int64_t)(r0 + r) * io.in_row + c0 + c];
            }
            v = (float)((double)v * scale);
        }
        if (g.trans) sub.at[c][r] = v;
        else sub.at[r][c] = v;
    }
    wave_sync();
    char* x = ws + g.x + ((int64_t)idx * cells + (int64_t)ci * g.sn + cj) * CELL;
    char* xt = ws + g.xt[0] + ((int64_t)idx * cells + (int64_t)cj * g.sm + ci) * CELL;
    float v[8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        sub.rows(q, lane, v);
        store_terms(x, q, lane, v);
        sub.columns(q, lane, v);
        store_terms(xt, q, lane, v);
    }
}

// ---- products --------------------------------------------------------------------------------------------------------------
// one wave's 1 KB from memory to LDS: lane l's 16 bytes at src land at dst + 16 l (dst is the same in every lane).  The
// load is in flight when this returns: the ring below waits for it by count.
__device__ __forceinline__ void piece_to_lds(const char* src, unsigned dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(src), "s"(dst) : "memory");
}

enum { MAKE_S, MAKE_R, MAKE_X, MAKE_LAST };              // S = X X^T; R = b S + c S S; X = a X + R X; the same, result out
enum { OUT_F32, OUT_BF16, OUT_F16, OUT_MUON };

// TI x TJ cells a workgroup, WI x WJ waves, a ring of RING k blocks in LDS
template <int TI, int TJ, int WI, int WJ, int RING, int WHAT, int OUT>
__global__ __launch_bounds__(WI * WJ * 64) void orth_product_kernel(Plan plan, Pointers ptr, Ends io, int to, char* __restrict__ ws) {
    constexpr int W = WI * WJ, FI = TI / WI, FJ = TJ / WJ;
    constexpr int STAGE = (TI + TJ) * 2 * PIECE, LOADS = (TI + TJ) * 2 / W;
    static_assert((TI + TJ) * 2 % W == 0 && TI % WI == 0 && TJ % WJ == 0, "whole pieces and cells per wave");
    static_assert(W * 32 * 33 * 4 <= RING * STAGE, "the epilogue reuses the ring");
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile = xcd_order(blockIdx.x, gridDim.x);
    int k = 0;
    while (k + 1 < plan.groups && tile >= plan.first_tile[k + 1]) ++k;
    const Group& g = plan.g[k];
    // the tile's cells
    constexpr bool SYM = WHAT == MAKE_S || WHAT == MAKE_R;
    const int ni = (g.sm + TI - 1) / TI, nj = SYM ? ni : (g.sn + TJ - 1) / TJ;
    const int per = SYM ? ni * (ni + 1) / 2 : ni * nj;
    const int in_group = tile - plan.first_tile[k], idx = in_group / per;
    int t = in_group - idx * per, ti, tj;
    if (SYM) {                                           // the triangle tj >= ti, row by row
        ti = 0;
        while (t >= ni - ti) t -= ni - ti++;
        tj = ti + t;
    } else {
        ti = t / nj;
        tj = t - ti * nj;
    }
    const int64_t xm = (int64_t)idx * g.sm * g.sn * CELL, sm2 = (int64_t)idx * g.sm * g.sm * CELL;
    const int cur = to ^ 1;
    const char* p = ws + (WHAT == MAKE_S ? g.x + xm : WHAT == MAKE_R ? g.s + sm2 : g.r + sm2);
    const char* q = ws + (WHAT == MAKE_S ? g.x + xm : WHAT == MAKE_R ? g.s + sm2 : g.xt[cur] + xm);
    const int kcells = WHAT == MAKE_S ? g.sn : g.sm, steps = 2 * kcells;
    const int prows = g.sm, qrows = SYM ? g.sm : g.sn;

    // this wave's pieces of a k block: cells past the matrix read its last ones (their results are not kept)
    const char* src[LOADS];
    unsigned dst[LOADS];
    const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
#pragma unroll
    for (int l = 0; l < LOADS; ++l) {
        const int piece = wave * LOADS + l, cell = piece >> 1, term = piece & 1;
        int row = cell < TI ? ti * TI + cell : tj * TJ + cell - TI;
        const int most = (cell < TI ? prows : qrows) - 1;
        row = row < most ? row : most;
        src[l] = (cell < TI ? p : q) + (int64_t)row * kcells * CELL + term * PIECE + lane * 16;
        dst[l] = base + piece * PIECE;
    }
    int filled = 0;                                      // k blocks requested so far
    auto fill = [&]() {
        const unsigned at = (unsigned)(filled % RING) * STAGE;
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            piece_to_lds(src[l], dst[l] + at);
            src[l] += 2 * PIECE;
        }
        ++filled;
    };
    f32x16 acc[FI][FJ];
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    const int wi = wave / WJ, wj = wave - wi * WJ;
    while (filled < RING - 1 && filled < steps) fill();
    for (int s = 0; s < steps; ++s) {
        // block s has landed when at most the blocks behind it are still on their way (loads return in order); then every
        // wave is past its reads of block s - 1, whose place block s + RING - 1 takes
        if (filled - s == RING - 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RING - 2) * LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (filled < steps) fill();
        const char* stage = lds + (s % RING) * STAGE + lane * 16;
        f16x8 a[FI][2], b[FJ][2];
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) a[i][h] = *reinterpret_cast<const f16x8*>(stage + ((wi * FI + i) * 2 + h) * PIECE);
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) b[j][h] = *reinterpret_cast<const f16x8*>(stage + ((TI + wj * FJ + j) * 2 + h) * PIECE);
#pragma unroll
        for (int term = 0; term < 3; ++term)
#pragma unroll
            for (int i = 0; i < FI; ++i)
#pragma unroll
                for (int j = 0; j < FJ; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][term == 1], b[j][term == 0], acc[i][j], 0, 0, 0);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // the ring becomes the epilogue's

    const Sub sub = {reinterpret_cast<float(*)[33]>(lds + wave * 32 * 33 * 4)};
    float rate = 0.f;
    if (WHAT == MAKE_LAST && OUT == OUT_MUON) {
        const float rows = (float)(g.trans ? g.n : g.m), cols = (float)(g.trans ? g.m : g.n);
        rate = io.lr * sqrtf(fmaxf(1.f, rows / cols));
    }
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
            const int ci = ti * TI + wi * FI + i, cj = tj * TJ + wj * FJ + j;
            if (ci >= prows || cj >= qrows) continue;
            wave_sync();                                 // (the cell before this one has been read)
#pragma unroll
            for (int r = 0; r < 16; ++r) sub.at[8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)][lane & 31] = acc[i][j][r];
            wave_sync();
            float v[8], w[8];
            if constexpr (SYM) {
                char* out = ws + (WHAT == MAKE_S ? g.s : g.r) + sm2;
                const char* s = ws + g.s + sm2;
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    if (side && ti == tj) break;         // (a tile on the diagonal holds both halves)
                    const int64_t at = ((int64_t)(side ? cj : ci) * g.sm + (side ? ci : cj)) * CELL;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (side) sub.columns(h, lane, v);
                        else sub.rows(h, lane, v);
                        if (WHAT == MAKE_S) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] *= 0x1p-15f;
                        } else {
                            load_terms(s + at, h, lane, w);
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] = (CB * 0x1p-1f) * w[e] + (CC * 0x1p-16f) * v[e];
                        }
                        store_terms(out + at, h, lane, v);
                    }
                }
            } else {
                char* x = ws + g.x + xm + ((int64_t)ci * g.sn + cj) * CELL;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    sub.rows(h, lane, v);
                    load_terms(x, h, lane, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = CA * w[e] + 0x1p-14f * v[e];
                    sub.put_rows(h, lane, v);
                    if (WHAT == MAKE_X) store_terms(x, h, lane, v);
                }
                wave_sync();
                if constexpr (WHAT == MAKE_X) {
                    char* xt = ws + g.xt[to] + xm + ((int64_t)cj * g.sm + ci) * CELL;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        sub.columns(h, lane, v);
                        store_terms(xt, h, lane, v);
                    }
                } else {
                    const int mat = g.first + idx;
                    const int r0 = (g.trans ? cj : ci) * 32, c0 = (g.trans ? ci : cj) * 32;
                    const int rows = g.trans ? g.n : g.m, cols = g.trans ? g.m : g.n;
#pragma unroll
                    for (int it = 0; it < 16; ++it) {
                        const int r = it * 2 + (lane >> 5), c = lane & 31;
                        if (r0 + r >= rows || c0 + c >= cols) continue;
                        const float o = (g.trans ? sub.at[c][r] : sub.at[r][c]) * 0x1p-15f;
                        if constexpr (OUT == OUT_MUON) {
                            float* w0 = ptr.param[mat] + (int64_t)(r0 + r) * cols + c0 + c;
                            *w0 = __builtin_fmaf(-rate, o, *w0 * io.keep);
                        } else {
                            const int64_t at = mat * io.out_matrix + (int64_t)(r0 + r) * io.out_row + c0 + c;
                            if (OUT == OUT_F32) ((float*)io.out)[at] = o;
                            else if (OUT == OUT_BF16) ((__bf16*)io.out)[at] = (__bf16)o;
                            else ((_Float16*)io.out)[at] = (_Float16)o;
                        }
                    }
                }
            }
        }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
inline int cells_of(int64_t n) { return (int)((n + 31) / 32); }

// workspace: partial sums of the norms, then each group's X, X^T (two), S, R
size_t layout(Plan& plan, int matrices) {
    int64_t at = (int64_t)matrices * NORM_BLOCKS * sizeof(double);
    for (int k = 0; k < plan.groups; ++k) {
        Group& g = plan.g[k];
        const int64_t x = (int64_t)g.count * g.sm * g.sn * CELL, s = (int64_t)g.count * g.sm * g.sm * CELL;
        g.x = at;
        g.xt[0] = at + x;
        g.xt[1] = at + 2 * x;
        g.s = at + 3 * x;
        g.r = g.s + s;
        at = g.r + s;
    }
    return (size_t)at;
}

Group group_of(int rows, int cols, int count, int first) {
    Group g = {};
    g.trans = rows > cols;
    g.m = g.trans ? cols : rows;
    g.n = g.trans ? rows : cols;
    g.sm = cells_of(g.m);
    g.sn = cells_of(g.n);
    g.count = count;
    g.first = first;
    return g;
}

// first_tile of a launch with TI x TJ cells a workgroup; the number of workgroups, or -1 where they do not fit a grid
int64_t count_tiles(Plan& plan, int t, bool sym) {
    int64_t total = 0;
    for (int k = 0; k < plan.groups; ++k) {
        const Group& g = plan.g[k];
        const int64_t ni = (g.sm + t - 1) / t, nj = (g.sn + t - 1) / t;
        plan.first_tile[k] = (int)total;
        total += g.count * (sym ? ni * (ni + 1) / 2 : ni * nj);
        if (total > 0x7fffffff) return -1;
    }
    plan.first_tile[plan.groups] = (int)total;
    return total;
}

template <int T, int WI, int WJ, int RING, int WHAT, int OUT>
int launch_product(const Plan& plan, const Pointers& ptr, const Ends& io, int to, int64_t tiles, char* ws, hipStream_t stream) {
    constexpr size_t lds = (size_t)RING * T * 4 * PIECE;
    static unsigned long long done;
    if (lds > 64 * 1024) {
        const int e = nf_raise_lds_cap((const void*)orth_product_kernel<T, T, WI, WJ, RING, WHAT, OUT>, &done);
        if (e) return e;
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_product_kernel<T, T, WI, WJ, RING, WHAT, OUT>), dim3((unsigned)tiles),
                       dim3(WI * WJ * 64), lds, stream, plan, ptr, io, to, ws);
    return nf_launch_status();
}

template <int WHAT, int OUT>
int product(Plan& plan, const Pointers& ptr, const Ends& io, int to, char* ws, hipStream_t stream) {
    // the largest tile that still gives most of the 256 CUs one
    constexpr bool SYM = WHAT == MAKE_S || WHAT == MAKE_R;
    int64_t tiles = count_tiles(plan, 8, SYM);
    if (tiles >= 128) return launch_product<8, 2, 4, 4, WHAT, OUT>(plan, ptr, io, to, tiles, ws, stream);
    tiles = count_tiles(plan, 4, SYM);
    if (tiles >= 128) return launch_product<4, 2, 2, 3, WHAT, OUT>(plan, ptr, io, to, tiles, ws, stream);
    tiles = count_tiles(plan, 2, SYM);
    if (tiles < 0) return NF_ERR_SHAPE;
    return launch_product<2, 2, 2, 4, WHAT, OUT>(plan, ptr, io, to, tiles, ws, stream);
}

template <typename T, bool MUON, int OUT>
int run(Plan& plan, const Pointers& ptr, const Ends& io, int matrices, int steps, double eps, void* workspace, hipStream_t stream) {
    char* ws = (char*)workspace;
    double* partial = (double*)workspace;
    int64_t most = 1;
    for (int k = 0; k < plan.groups; ++k) {
        const int64_t size = (int64_t)plan.g[k].m * plan.g[k].n;
        most = size > most ? size : most;
    }
    int64_t blocks = (most + 4095) / 4096;
    if (blocks > NORM_BLOCKS) blocks = NORM_BLOCKS;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_norm_kernel<T, MUON>), dim3((unsigned)blocks, (unsigned)matrices), dim3(256), 0, stream,
                       plan, ptr, io, partial);
    int e = nf_launch_status();
    if (e) return e;
    int64_t total = 0;
    for (int k = 0; k < plan.groups; ++k) {
        plan.first_tile[k] = (int)total;
        total += (int64_t)plan.g[k].count * (((int64_t)plan.g[k].sm * plan.g[k].sn + 3) / 4);
        if (total > 0x7fffffff) return NF_ERR_SHAPE;
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_start_kernel<T, MUON>), dim3((unsigned)total), dim3(256), 0, stream, plan, ptr, io,
                       partial, (int)blocks, eps, ws);
    if ((e = nf_launch_status())) return e;
    for (int s = 0; s < steps; ++s) {
        const int to = (s + 1) & 1;
        if ((e = product<MAKE_S, OUT_F32>(plan, ptr, io, to, ws, stream))) return e;
        if ((e = product<MAKE_R, OUT_F32>(plan, ptr, io, to, ws, stream))) return e;
        if (s + 1 < steps) e = product<MAKE_X, OUT_F32>(plan, ptr, io, to, ws, stream);
        else e = product<MAKE_LAST, OUT>(plan, ptr, io, to, ws, stream);
        if (e) return e;
    }
    return NF_OK;
}

constexpr int MAX_MATRIX_GRID = 65535;   // matrices of one call (a grid's y extent)
constexpr int MAX_SIDE = 1 << 20;

bool sizes_ok(int64_t count, int rows, int cols) {
    return count >= 0 && count <= MAX_MATRIX_GRID && rows >= 1 && cols >= 1 && rows <= MAX_SIDE && cols <= MAX_SIDE;
}

// The matrices from `from` on that one sequence of launches takes, grouped by shape: `order` lists them group by group.
// Returns how many.
int plan_muon(const int* rows, const int* cols, int from, int count, Plan& plan, int* order) {
    int taken = 0, shapes[MAX_GROUPS][2], groups = 0, of[MAX_MATRICES];
    while (from + taken < count && taken < MAX_MATRICES) {
        const int r = rows[from + taken], c = cols[from + taken];
        int k = 0;
        while (k < groups && (shapes[k][0] != r || shapes[k][1] != c)) ++k;
        if (k == groups) {
            if (groups == MAX_GROUPS) break;
            shapes[k][0] = r;
            shapes[k][1] = c;
            ++groups;
        }
        of[taken++] = k;
    }
    int at = 0;
    plan.groups = groups;
    for (int k = 0; k < groups; ++k) {
        const int first = at;
        for (int i = 0; i < taken; ++i)
            if (of[i] == k) order[at++] = from + i;
        plan.g[k] = group_of(shapes[k][0], shapes[k][1], at - first, first);
    }
    return taken;
}

}  // namespace

extern "C" size_t nf_orthogonalize_workspace_bytes(int64_t count, int rows, int cols) {
    if (!sizes_ok(count, rows, cols) || count == 0) return 0;
    Plan plan = {};
    plan.groups = 1;
    plan.g[0] = group_of(rows, cols, (int)count, 0);
    return layout(plan, (int)count);
}

extern "C" int nf_orthogonalize(const void* matrices, int64_t matrix_stride, int64_t row_stride, void* out,
                                int64_t out_matrix_stride, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                                int64_t count, int rows, int cols, int steps, double eps, int elem, void* stream) {
    const int size = nf_elem_size(elem);
    if (!size) return NF_ERR_DTYPE;
    if (!sizes_ok(count, rows, cols) || steps < 1 || !(eps >= 0.0)) return NF_ERR_SHAPE;
    if (count == 0) return NF_OK;
    if (!matrices || !out || !workspace) return NF_ERR_NULL;
    if (matrix_stride < 0 || row_stride < 0 || (rows > 1 && out_row_stride < cols) ||
        (count > 1 && out_matrix_stride < (rows - 1) * out_row_stride + cols) || !nf_aligned(matrices, size) ||
        !nf_aligned(out, size) || !nf_aligned(workspace, 16))
        return NF_ERR_LAYOUT;
    Plan plan = {};
    plan.groups = 1;
    plan.g[0] = group_of(rows, cols, (int)count, 0);
    if (workspace_bytes < layout(plan, (int)count)) return NF_ERR_SCRATCH;
    Pointers ptr = {};
    Ends io = {};
    io.in = matrices;
    io.out = out;
    io.in_matrix = matrix_stride;
    io.in_row = row_stride;
    io.out_matrix = out_matrix_stride;
    io.out_row = out_row_stride;
    hipStream_t s = (hipStream_t)stream;
    if (elem == NF_ELEM_F32) return run<float, false, OUT_F32>(plan, ptr, io, (int)count, steps, eps, workspace, s);
    if (elem == NF_ELEM_BF16) return run<__bf16, false, OUT_BF16>(plan, ptr, io, (int)count, steps, eps, workspace, s);
    return run<_Float16, false, OUT_F16>(plan, ptr, io, (int)count, steps, eps, workspace, s);
}

extern "C" size_t nf_muon_workspace_bytes(const int* rows, const int* cols, int count) {
    if (!rows || !cols) return 0;
    size_t most = 0;
    int order[MAX_MATRICES];
    for (int at = 0; at < count;) {
        for (int i = at; i < count && i < at + MAX_MATRICES; ++i)
            if (!sizes_ok(1, rows[i], cols[i])) return 0;
        Plan plan = {};
        const int taken = plan_muon(rows, cols, at, count, plan, order);
        const size_t need = layout(plan, taken);
        most = need > most ? need : most;
        at += taken;
    }
    return most;
}

extern "C" int nf_muon_update(float* const* params, const float* const* grads, float* const* momenta, const int* rows,
                              const int* cols, int count, double lr, double momentum, int nesterov, double weight_decay,
                              int steps, double eps, void* workspace, size_t workspace_bytes, void* stream) {
    if (count < 0 || steps < 1 || !(eps >= 0.0)) return NF_ERR_SHAPE;
    if (count == 0) return NF_OK;
    if (!params || !grads || !momenta || !rows || !cols || !workspace) return NF_ERR_NULL;
    for (int i = 0; i < count; ++i) {
        if (!sizes_ok(1, rows[i], cols[i])) return NF_ERR_SHAPE;
        if (!params[i] || !grads[i] || !momenta[i]) return NF_ERR_NULL;
        if (!nf_aligned(params[i], 4) || !nf_aligned(grads[i], 4) || !nf_aligned(momenta[i], 4)) return NF_ERR_LAYOUT;
    }
    if (!nf_aligned(workspace, 16)) return NF_ERR_LAYOUT;
    if (workspace_bytes < nf_muon_workspace_bytes(rows, cols, count)) return NF_ERR_SCRATCH;
    int order[MAX_MATRICES];
    for (int at = 0; at < count;) {
        Plan plan = {};
        const int taken = plan_muon(rows, cols, at, count, plan, order);
        layout(plan, taken);
        Pointers ptr = {};
        for (int i = 0; i < taken; ++i) {
            ptr.grad[i] = grads[order[i]];
            ptr.momentum[i] = momenta[order[i]];
            ptr.param[i] = params[order[i]];
        }
        Ends io = {};
        io.momentum = (float)momentum;
        io.nesterov = nesterov;
        io.keep = (float)(1.0 - lr * weight_decay);
        io.lr = (float)lr;
        const int e = run<float, true, OUT_MUON>(plan, ptr, io, taken, steps, eps, workspace, (hipStream_t)stream);
        if (e) return e;
        at += taken;
    }
    return NF_OK;
}
