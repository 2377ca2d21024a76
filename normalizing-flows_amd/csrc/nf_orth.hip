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
// their elements times 2^15, 2^15 and 2^14 fit fp16, and lo keeps its bits down to 2^-39 of 1: fixed scales, no searches.
// That is enough for S and b S + c S S, which stand beside the identity.  X alone can be small throughout, where |G| is far
// below eps: its scale is 2^(15 + raise), `raise` the whole powers of two that |X| is known to lie below 1 - taken from the
// norm for X0, less the growth of at most a factor a in every step after it (0 throughout for |G| >= eps).
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
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr double DA = 3.4445, DB = -4.7750, DC = 2.0315;
constexpr float CA = 3.4445f, CB = -4.7750f, CC = 2.0315f;
constexpr int CELL = 4096;               // bytes of a 32 x 32 cell
constexpr int PIECE = 1024;              // of one term of one 32 x 16 block
constexpr int MAX_GROUPS = 8;            // shapes in one sequence of launches
constexpr int MAX_MATRICES = 48;         // matrices with pointers of their own (kernel arguments) in one sequence
constexpr int NORM_STRIDE = 256;         // doubles of a matrix in the workspace's first part: ...
constexpr int NORM_BLOCKS = NORM_STRIDE - 1;             // ... partial sums of its norm, and X0's raise
constexpr int NORM_THREADS = 512;        // of its workgroups (4096 x 1024: 354 us, with 256 363; with 1024 level: 352 there, 20 of
                                         // 512 x 512 332 instead of 329; three runs of each in turn on one device)
constexpr int64_t SEQUENCE_BYTES = (int64_t)8 << 30;     // of X's and the slots' cells of one sequence of more than one matrix

// matrices of one shape
struct Group {
    int m, n;                            // m <= n
    int sm, sn;                          // cells along each
    int trans;                           // rows > columns: X = G^T
    int count, first;                    // matrices, index of the first
    int64_t x, xt0, xt1, s;               // byte offsets in the workspace: X, X^T (two), the slots of m x m matrices, each
                                         // of them `count` matrices one behind the other
};
struct Plan {
    Group g[MAX_GROUPS];
    int first_tile[MAX_GROUPS + 1];      // workgroups of the launch, group by group
    int parts[MAX_GROUPS];               // of the k cells of a symmetric product's tile
    int64_t partial[MAX_GROUPS];         // offset of their accumulators, in floats
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

// 1 / (norm + eps), finite for a zero matrix over the smallest eps too (zeros stay zeros; with eps = 0 they are NaN)
__device__ __forceinline__ double over_norm(double norm, double eps) {
    const double d = norm + eps;
    return 1.0 / (d > 0 && d < 1e-290 ? 1e-290 : d);
}
// X0's raise: 2^raise <= (norm + eps) / norm = 1 / |X0|
__device__ __forceinline__ int raise_of(double norm, double eps) {
    if (!(norm > 0) || !(norm + eps < INFINITY)) return 0;
    const int e = ilogb(norm + eps) - ilogb(norm) - 1;
    return e > 0 ? e : 0;
}
// ... and X's after `done` steps: a < 2^(457 / 256)
__device__ __forceinline__ int raise_after(int first, int done) {
    const int64_t less = ((int64_t)done * 457 + 255) >> 8;
    return first > less ? (int)(first - less) : 0;
}
// where the workspace keeps it for the launches after the first two
__device__ __forceinline__ int raise_in(const double* norms, int mat) {
    return *reinterpret_cast<const int*>(norms + (int64_t)mat * NORM_STRIDE + NORM_BLOCKS);
}

// (LDS traffic of a wave with itself: in order, but only this tells the compiler that lanes talk to each other)
__device__ __forceinline__ void wave_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Workgroups go round robin to the eight XCDs, each with an L2 of its own: XCD k gets the k-th eighth of a group's tiles.
__device__ __forceinline__ int xcd_order(int id, int total) {
    const int q = total >> 3, rest = total & 7, xcd = id & 7;
    return xcd * q + (xcd < rest ? xcd : rest) + (id >> 3);
}

// ---- norm and momentum -------------------------------------------------------------------------------------------------
// partial[matrix][block] = sum of squares in fp64 (no overflow or underflow over the whole fp32 range, and the same bits
// every time); MUON: momentum <- mu momentum + grad on the way, the norm is that of the update
template <typename T, bool MUON>
__global__ __launch_bounds__(NORM_THREADS) void orth_norm_kernel(Plan plan, Pointers ptr, Ends io, double* __restrict__ partial) {
    __shared__ double red[NORM_THREADS / 64];
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
        constexpr int EACH = 4;                          // (loads before the first store: their latency is paid once)
        for (int64_t e0 = (int64_t)blockIdx.x * (EACH * NORM_THREADS) + threadIdx.x; e0 < total; e0 += (int64_t)blocks * (EACH * NORM_THREADS)) {
            float gv[EACH], mv[EACH];
#pragma unroll
            for (int l = 0; l < EACH; ++l) {
                const int64_t e = e0 + l * NORM_THREADS;
                gv[l] = e < total ? gr[e] : 0.f;
                mv[l] = e < total ? mo[e] : 0.f;
            }
#pragma unroll
            for (int l = 0; l < EACH; ++l) {
                const int64_t e = e0 + l * NORM_THREADS;
                const float v = __builtin_fmaf(io.momentum, mv[l], gv[l]);
                if (e < total) mo[e] = v;
                const double u = io.nesterov ? __builtin_fmaf(io.momentum, v, gv[l]) : v;
                sum += u * u;
            }
        }
    } else {
        const T* in = (const T*)io.in + mat * io.in_matrix;
        const int rows = g.trans ? g.n : g.m;
        constexpr int ROWS = 4, EACH = 2;                // (their loads together on their way)
        for (int64_t row0 = blockIdx.x; row0 < rows; row0 += (int64_t)ROWS * blocks)
            for (int c0 = threadIdx.x; c0 < cols; c0 += EACH * NORM_THREADS) {
                float v[ROWS][EACH];
#pragma unroll
                for (int i = 0; i < ROWS; ++i)
#pragma unroll
                    for (int l = 0; l < EACH; ++l) {
                        const int64_t row = row0 + (int64_t)i * blocks;
                        const int c = c0 + l * NORM_THREADS;
                        v[i][l] = row < rows && c < cols ? (float)in[row * io.in_row + c] : 0.f;
                    }
#pragma unroll
                for (int i = 0; i < ROWS; ++i)
#pragma unroll
                    for (int l = 0; l < EACH; ++l) sum += (double)v[i][l] * v[i][l];
            }
    }
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0;
        for (int w = 0; w < NORM_THREADS / 64; ++w) sum += red[w];
        partial[(int64_t)mat * NORM_STRIDE + blockIdx.x] = sum;
    }
}

// ---- cells ---------------------------------------------------------------------------------------------------------------
// A value's two terms.  The empty asm makes v one rounded number: where it is a product, the compiler may otherwise round
// the exact product to hi in one place and v in another, and where these differ (once in some 2^13 values) hi + lo is off by
// a step of hi.
__device__ __forceinline__ void split(float v, _Float16& hi, _Float16& lo) {
    asm("" : "+v"(v));
    hi = (_Float16)v;
    lo = (_Float16)(v - (float)hi);
}

// both in a word, hi in the low half
__device__ __forceinline__ uint32_t split(float v) {
    _Float16 hi, lo;
    split(v, hi, lo);
    return (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
}

// A wave's 32 x 32 words in LDS: values change between the layout of the accumulators (or of the caller's matrix) and the
// two orientations of a cell.
struct Sub {
    uint32_t (*at)[33];
    // this lane's part of the cell (row lane % 32, columns 16 q + 8 (lane / 32) ..), or of its transpose, to memory
    template <bool TRANSPOSED>
    __device__ __forceinline__ void store(char* cell, int lane) const {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int r = lane & 31, c = 16 * q + 8 * (lane >> 5);
            u32x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t v = TRANSPOSED ? at[c + 2 * e][r] : at[r][c + 2 * e];
                const uint32_t w = TRANSPOSED ? at[c + 2 * e + 1][r] : at[r][c + 2 * e + 1];
                hi[e] = (v & 0xffff) | w << 16;
                lo[e] = v >> 16 | (w & 0xffff0000);
            }
            *reinterpret_cast<u32x4*>(cell + q * 2 * PIECE + lane * 16) = hi;
            *reinterpret_cast<u32x4*>(cell + q * 2 * PIECE + PIECE + lane * 16) = lo;
        }
    }
};

// X0 in both orientations: a wave a cell
template <typename T, bool MUON>
__global__ __launch_bounds__(256) void orth_start_kernel(Plan plan, Pointers ptr, Ends io, double* partial,
                                                         int blocks, double eps, char* __restrict__ ws) {
    __shared__ uint32_t lds[4][32][33];
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
    for (int e = lane; e < blocks; e += 64) sum += partial[(int64_t)mat * NORM_STRIDE + e];
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    const int raise = raise_of(sqrt(sum), eps);
    if (cell == 0 && lane == 0) *reinterpret_cast<int*>(partial + (int64_t)mat * NORM_STRIDE + NORM_BLOCKS) = raise;
    const double scale = ldexp(over_norm(sqrt(sum), eps), raise + 15);
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
        if (g.trans) sub.at[c][r] = split(v);
        else sub.at[r][c] = split(v);
    }
    wave_sync();
    char* x = ws + g.x + ((int64_t)idx * cells + (int64_t)ci * g.sn + cj) * CELL;
    char* xt = ws + g.xt0 + ((int64_t)idx * cells + (int64_t)cj * g.sm + ci) * CELL;
    sub.store<false>(x, lane);
    sub.store<true>(xt, lane);
}

// ---- products --------------------------------------------------------------------------------------------------------------
// one wave's 1 KB from memory to LDS: lane l's 16 bytes at src land at dst + 16 l (dst is the same in every lane).  The
// load is in flight when this returns: the ring below waits for it by count.
__device__ __forceinline__ void piece_to_lds(const char* src, unsigned dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(src), "s"(dst) : "memory");
}

// A symmetric result in slot `out`: k0 (P Q^T + k1 E1 + k2 E2), the factors with the powers of two of the operands' scales
// (P = Q = X where p is FROM_X, else slots; E1, E2: slots or NONE).  The E's join the accumulators when the product is
// complete: an accumulator that started from them would round every one of its 3 K / 16 sums at their size (measured: twice
// the error of the whole iteration).
constexpr int FROM_X = -1, NONE = -1;
struct SymOp { int p, q, out, e1, e2; float k0, k1, k2; };
struct SymOps { SymOp op[2]; int done; };                // `done`: steps that X has gone through (FROM_X)
// X <- alpha X + T X from slot r: the accumulators get scale_x * X (alpha with T's power of two), and out_scale takes them
// back to X's scale; `done` and `after`: the steps that X has gone through before and after it
struct MixOp { int r, to; float scale_x, out_scale; int done, after; };

// vmcnt(N) lgkmcnt(0): at most N loads on their way, all LDS reads back
template <int N> __device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (0 << 8) | ((N >> 4) << 14));
}

// The k loop: TI x TJ cells, four waves in 2 x 2, each FI x FJ cells of 32 x 32.  A ring of RING k blocks of 16 in LDS.  Step s
// multiplies block s from registers and meanwhile reads block s + 1 from LDS into a second set of fragments and requests
// block s + RING into the place of block s: reads and requests go between the matrix instructions, which a single wave per
// SIMD must issue without a pause.  `p`, `q`: the operands' cells of row 0; rows past the matrix read its last ones (their
// results are not kept).
template <int TI, int TJ, int RING>
struct Ring {
    static constexpr int FI = TI / 2, FJ = TJ / 2, STAGE = (TI + TJ) * 2 * PIECE, LOADS = (TI + TJ) / 2;
    static constexpr int READS = 2 * (FI + FJ);
    f32x16 acc[FI][FJ];
    f16x8 frag_a[2][FI][2], frag_b[2][FJ][2];            // [set][cell][term]
    const char* src[LOADS];
    unsigned dst[LOADS];
    unsigned place;                                      // of the next request
    const char *from_a, *from_b;                         // this lane's fragments in place 0
    unsigned next;                                       // place of the next block to read

    __device__ __forceinline__ void request(int l) {
        piece_to_lds(src[l], dst[l] + place);
        src[l] += 2 * PIECE;
    }
    __device__ __forceinline__ void turn(unsigned& at) { at = at == (RING - 1) * STAGE ? 0 : at + STAGE; }
    __device__ __forceinline__ void fill() {
#pragma unroll
        for (int l = 0; l < LOADS; ++l) request(l);
        turn(place);
    }
    __device__ __forceinline__ void read(int set, int r) {                       // fragment r of READS
        if (r < 2 * FI) frag_a[set][r >> 1][r & 1] = *reinterpret_cast<const f16x8*>(from_a + next + r * PIECE);
        else frag_b[set][(r >> 1) - FI][r & 1] = *reinterpret_cast<const f16x8*>(from_b + next + (r - 2 * FI) * PIECE);
    }
    // one step: FILL requests a block, READ reads the next one
    template <int SET, bool FILL, bool READ>
    __device__ __forceinline__ void step() {
        constexpr int M = 3 * FI * FJ, EACH = (READS * 3 + 2 * M - 1) / (2 * M), PER = M / LOADS;
        int r = 0, l = 0;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const int term = m / (FI * FJ), i = m / FJ % FI, j = m % FJ;
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(frag_a[SET][i][term == 1], frag_b[SET][j][term == 0], acc[i][j], 0, 0, 0);
            if (READ && r < READS) {                     // within the first two thirds of the products
#pragma unroll
                for (int e = 0; e < EACH; ++e)
                    if (r < READS) read(SET ^ 1, r++);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (FILL && (m + 1) % PER == 0 && l < LOADS) {
                request(l++);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (FILL) {
#pragma unroll
            for (int e = M / PER; e < LOADS; ++e) request(e);
            turn(place);
        }
        if (READ) turn(next);
    }
    // block s + 1 has landed when at most N requests behind it are on their way (loads return in order), and this wave's
    // reads of block s are back; the barrier makes that true of all four waves
    template <int N> __device__ __forceinline__ void meet() {
        asm volatile("" ::: "memory");
        wait_loads<N>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    }
    // E of this wave's cells in the accumulators' layout, from the cells of E^T (rows as Q's, columns as P's): an
    // accumulator's four rows are 8 bytes there
    struct Terms { f16x4 v[FI][FJ][4][2]; };
    __device__ __forceinline__ void load(Terms& t, const char* et, int64_t row_bytes, int ci0, int cj0, int prows, int qrows) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j) {
                const int ci = ci0 + i < prows ? ci0 + i : prows - 1, cj = cj0 + j < qrows ? cj0 + j : qrows - 1;
                const char* cell = et + cj * row_bytes + (int64_t)ci * CELL + (lane & 31) * 16 + (lane >> 5) * 8;
#pragma unroll
                for (int g = 0; g < 4; ++g)              // rows 8 g + 4 (lane / 32) .. + 3
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        t.v[i][j][g][h] = *reinterpret_cast<const f16x4*>(cell + (g >> 1) * 2 * PIECE + (g & 1) * 512 + h * PIECE);
            }
    }
    __device__ __forceinline__ void add(const Terms& t, float scale) {
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j)
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[i][j][4 * g + e] = __builtin_fmaf(scale, (float)t.v[i][j][g][0][e] + (float)t.v[i][j][g][1][e], acc[i][j][4 * g + e]);
    }
    // k cells first .. last - 1 (at least one); `ahead` is called where all blocks have been requested, for what the epilogue
    // wants to have by then
    template <typename Ahead>
    __device__ __forceinline__ void run(char* lds, const char* p, const char* q, int64_t row_bytes, int ti, int tj, int prows,
                                        int qrows, int first, int last, Ahead ahead) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int wi = wave >> 1, wj = wave & 1;
        const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            const int piece = wave * LOADS + l, cell = piece >> 1, term = piece & 1;
            int row = cell < TI ? ti * TI + cell : tj * TJ + cell - TI;
            const int most = (cell < TI ? prows : qrows) - 1;
            row = row < most ? row : most;
            src[l] = (cell < TI ? p : q) + row * row_bytes + (int64_t)first * CELL + term * PIECE + lane * 16;
            dst[l] = base + piece * PIECE;
        }
        from_a = lds + wi * FI * 2 * PIECE + lane * 16;
        from_b = lds + (TI + wj * FJ) * 2 * PIECE + lane * 16;
        place = next = 0;
        const int steps = 2 * (last - first);            // even, at least 2
#pragma unroll
        for (int s = 0; s < RING; ++s)
            if (s < steps) fill();
        clear();
        if (steps > RING) meet<(RING - 1) * LOADS>();
        else meet<0>();
#pragma unroll
        for (int r = 0; r < READS; ++r) read(0, r);
        turn(next);
        int s = 0;
        for (; s + RING + 1 < steps; s += 2) {
            meet<(RING - 2) * LOADS>();
            step<0, true, true>();
            meet<(RING - 2) * LOADS>();
            step<1, true, true>();
        }
        if (RING % 2 && s + RING < steps) {              // (an odd ring's last request)
            meet<(RING - 2) * LOADS>();
            step<0, true, true>();
            meet<0>();
            step<1, false, true>();
            s += 2;
        }
        ahead();
        for (; s + 2 < steps; s += 2) {                  // the last blocks are all requested
            meet<0>();
            step<0, false, true>();
            meet<0>();
            step<1, false, true>();
        }
        meet<0>();
        step<0, false, true>();
        step<1, false, false>();
        meet<0>();                                       // the ring becomes the epilogue's
    }
};

// a cell's accumulators times `scale` into sub, as term pairs or as floats
template <bool TERMS>
__device__ __forceinline__ void put_acc(const Sub& sub, int lane, const f32x16& acc, float scale) {
    __builtin_amdgcn_sched_barrier(0);                   // (several cells' epilogues at once would not fit the registers)
    wave_sync();                                         // (what was there before has been read)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float v = acc[r] * scale;
        sub.at[8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)][lane & 31] = TERMS ? split(v) : __builtin_bit_cast(uint32_t, v);
    }
    wave_sync();
}

// one cell of a symmetric result at (ci, cj) and, where `mirror`, (cj, ci)
__device__ __forceinline__ void finish_sym(const Sub& sub, const f32x16& acc, float scale, char* out, int sm, int ci, int cj,
                                           bool mirror, int lane) {
    put_acc<true>(sub, lane, acc, scale);
    sub.store<false>(out + ((int64_t)ci * sm + cj) * CELL, lane);
    if (mirror) sub.store<true>(out + ((int64_t)cj * sm + ci) * CELL, lane);
}

// the triangle tj >= ti of n x n tiles, row by row
__device__ __forceinline__ void triangle(int t, int n, int& ti, int& tj) {
    ti = 0;
    while (t >= n - ti) t -= n - ti++;
    tj = ti + t;
}

// Symmetric products: blockIdx.y picks the operation.  Where a group's k cells are cut into parts (or `raw`), a workgroup takes
// one and leaves its raw accumulators in `partial`, which orth_sym_finish_kernel or orth_chain_kernel adds in order.
template <int T, int RING>
__global__ __launch_bounds__(256) void orth_sym_kernel(Plan plan, SymOps ops, int raw, const double* __restrict__ norms,
                                                       float* __restrict__ partial, char* __restrict__ ws) {
    extern __shared__ __align__(16) char lds[];
    const SymOp& op = ops.op[blockIdx.y];
    int k = 0;
    while (k + 1 < plan.groups && (int)blockIdx.x >= plan.first_tile[k + 1]) ++k;
    const Group& g = plan.g[k];
    const int n = (g.sm + T - 1) / T, per = n * (n + 1) / 2, parts = plan.parts[k];
    const int order = xcd_order(blockIdx.x - plan.first_tile[k], plan.first_tile[k + 1] - plan.first_tile[k]);
    // (a part's tiles are neighbours: they read the same rows)
    const int idx = order / (per * parts), in_matrix = order - idx * (per * parts), part = in_matrix / per, tile = in_matrix - part * per;
    int ti, tj;
    triangle(tile, n, ti, tj);
    const int64_t slot = (int64_t)g.count * g.sm * g.sm * CELL;
    char* slots = ws + g.s + (int64_t)idx * g.sm * g.sm * CELL;
    const bool from_x = op.p == FROM_X;
    const int raise = from_x ? raise_after(raise_in(norms, g.first + idx), ops.done) : 0;
    const char* p = from_x ? ws + g.x + (int64_t)idx * g.sm * g.sn * CELL : slots + op.p * slot;
    const char* q = from_x ? p : slots + op.q * slot;
    const int kcells = from_x ? g.sn : g.sm;
    const int first = (int)((int64_t)kcells * part / parts), last = (int)((int64_t)kcells * (part + 1) / parts);
    Ring<T, T, RING> ring;
    constexpr int F = T / 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave >> 1, wj = wave & 1;
    const int64_t row_bytes = (int64_t)kcells * CELL;
    typename Ring<T, T, RING>::Terms e;
    const bool has_e1 = op.e1 != NONE && part == 0, has_e2 = op.e2 != NONE && part == 0;
    ring.run(lds, p, q, row_bytes, ti, tj, g.sm, g.sm, first, last, [&]() {
        if (has_e1) ring.load(e, slots + op.e1 * slot, row_bytes, ti * T + wi * F, tj * T + wj * F, g.sm, g.sm);
    });
    if (has_e1) ring.add(e, op.k1);
    if (has_e2) {
        ring.load(e, slots + op.e2 * slot, row_bytes, ti * T + wi * F, tj * T + wj * F, g.sm, g.sm);
        ring.add(e, op.k2);
    }
    const Sub sub = {reinterpret_cast<uint32_t(*)[33]>(lds + wave * 32 * 33 * 4)};
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
            const int li = wi * F + i, lj = wj * F + j, ci = ti * T + li, cj = tj * T + lj;
            if (ci >= g.sm || cj >= g.sm) continue;
            if (parts > 1 || raw) {
                float* to = partial + plan.partial[k] +
                            ((((int64_t)blockIdx.y * g.count + idx) * per + tile) * parts + part) * (T * T * 1024) + (li * T + lj) * 1024 + lane * 4;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    *reinterpret_cast<float4*>(to + r * 256) = make_float4(ring.acc[i][j][4 * r], ring.acc[i][j][4 * r + 1],
                                                                           ring.acc[i][j][4 * r + 2], ring.acc[i][j][4 * r + 3]);
            } else {
                finish_sym(sub, ring.acc[i][j], ldexpf(op.k0, -2 * raise), slots + op.out * slot, g.sm, ci, cj, ti != tj, lane);
            }
        }
}

// a wave a cell: the partial accumulators of a tile's parts added in order, then the cell's epilogue (plan: the groups with
// parts only)
template <int T>
__global__ __launch_bounds__(256) void orth_sym_finish_kernel(Plan plan, SymOps ops, const double* __restrict__ norms,
                                                              const float* __restrict__ partial, char* __restrict__ ws) {
    __shared__ uint32_t lds[4][32][33];
    const SymOp& op = ops.op[blockIdx.y];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int k = 0;
    while (k + 1 < plan.groups && (int)blockIdx.x >= plan.first_tile[k + 1]) ++k;
    const Group& g = plan.g[k];
    const int n = (g.sm + T - 1) / T, per = n * (n + 1) / 2, parts = plan.parts[k];
    const int id = (blockIdx.x - plan.first_tile[k]) * 4 + wave, in_group = id / (T * T), local = id - in_group * (T * T);
    const int li = local / T, lj = local - li * T, idx = in_group / per;
    int ti, tj;
    triangle(in_group - idx * per, n, ti, tj);
    const int ci = ti * T + li, cj = tj * T + lj;
    if (ci >= g.sm || cj >= g.sm) return;                // (no barriers below: the waves are independent)
    const float* from = partial + plan.partial[k] +
                        (((int64_t)blockIdx.y * per * g.count + in_group) * parts * (T * T) + local) * 1024 + lane * 4;
    f32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0.f;
#pragma unroll 4
    for (int part = 0; part < parts; ++part, from += T * T * 1024) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float4 v = *reinterpret_cast<const float4*>(from + r * 256);
            acc[4 * r] += v.x;
            acc[4 * r + 1] += v.y;
            acc[4 * r + 2] += v.z;
            acc[4 * r + 3] += v.w;
        }
    }
    const Sub sub = {lds[wave]};
    const int64_t one = (int64_t)g.sm * g.sm * CELL;
    const int raise = op.p == FROM_X ? raise_after(raise_in(norms, g.first + idx), ops.done) : 0;
    finish_sym(sub, acc, ldexpf(op.k0, -2 * raise), ws + g.s + op.out * g.count * one + idx * one, g.sm, ci, cj, ti != tj, lane);
}

enum { OUT_X, OUT_F32, OUT_BF16, OUT_F16, OUT_MUON };

// X <- alpha X + T X: both orientations written (OUT_X), or the result in the caller's matrices
template <int TI, int TJ, int RING, int OUT>
__global__ __launch_bounds__(256, 2) void orth_mix_kernel(Plan plan, Pointers ptr, Ends io, MixOp op, const double* __restrict__ norms,
                                                          char* __restrict__ ws) {
    extern __shared__ __align__(16) char lds[];
    int k = 0;
    while (k + 1 < plan.groups && (int)blockIdx.x >= plan.first_tile[k + 1]) ++k;
    const Group& g = plan.g[k];
    const int ni = (g.sm + TI - 1) / TI, nj = (g.sn + TJ - 1) / TJ;
    const int in_group = xcd_order(blockIdx.x - plan.first_tile[k], plan.first_tile[k + 1] - plan.first_tile[k]);
    const int idx = in_group / (ni * nj), t = in_group - idx * (ni * nj);
    const int tj = t / ni, ti = t - tj * ni;             // (the tiles that share rows of X^T are neighbours)
    const int64_t xm = (int64_t)idx * g.sm * g.sn * CELL, slot = (int64_t)g.count * g.sm * g.sm * CELL;
    Ring<TI, TJ, RING> ring;
    constexpr int FI = TI / 2, FJ = TJ / 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave >> 1, wj = wave & 1;
    const int64_t row_bytes = (int64_t)g.sm * CELL;
    const char* xt = ws + (op.to ? g.xt0 : g.xt1) + xm;
    // X's own part from the rows of X^T that were Q's, from cache; with many cells a wave, only when the fragments are done
    typename Ring<TI, TJ, RING>::Terms e;
    auto own = [&]() { ring.load(e, xt, row_bytes, ti * TI + wi * FI, tj * TJ + wj * FJ, g.sm, g.sn); };
    ring.run(lds, ws + g.s + op.r * slot + (int64_t)idx * g.sm * g.sm * CELL, xt, row_bytes, ti, tj, g.sm, g.sn, 0, g.sm, [&]() {
        if (FI * FJ <= 4) own();
    });
    if (FI * FJ > 4) own();
    ring.add(e, op.scale_x);
    const Sub sub = {reinterpret_cast<uint32_t(*)[33]>(lds + wave * 32 * 33 * 4)};
    const int rows = g.trans ? g.n : g.m, cols = g.trans ? g.m : g.n, mat = g.first + idx;
    // back to X's scale after the step, or to 1 - in two factors, of which one alone may lie below fp32
    const int raise = raise_after(raise_in(norms, mat), op.done), most = raise < 64 ? raise : 64;
    const float back = ldexpf(op.out_scale, OUT == OUT_X ? raise_after(raise_in(norms, mat), op.after) - raise : -15 - most);
    const float rest = ldexpf(1.f, most - raise);
    const float rate = OUT == OUT_MUON ? io.lr * sqrtf(fmaxf(1.f, (float)rows / (float)cols)) * rest : 0.f;
    // four floats of a row of the caller's matrix a lane, where its rows allow it
    float* param = OUT == OUT_MUON ? ptr.param[mat] : nullptr;
    const bool wide = OUT == OUT_MUON && (cols & 3) == 0 && ((uintptr_t)param & 15) == 0;
#pragma unroll
    for (int i = 0; i < FI; ++i) {
        float4 old[FJ][4];
        if constexpr (OUT == OUT_MUON) {                 // (the row's parameters at once: their latency is paid once)
            if (wide) {
#pragma unroll
                for (int j = 0; j < FJ; ++j)
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        const int ci = ti * TI + wi * FI + i, cj = tj * TJ + wj * FJ + j;
                        const int r = (g.trans ? cj : ci) * 32 + it * 8 + (lane >> 3), c = (g.trans ? ci : cj) * 32 + (lane & 7) * 4;
                        old[j][it] = r < rows && c < cols ? *reinterpret_cast<const float4*>(param + (int64_t)r * cols + c)
                                                          : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
            }
        }
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
            const int ci = ti * TI + wi * FI + i, cj = tj * TJ + wj * FJ + j;
            if (ci >= g.sm || cj >= g.sn) continue;
            put_acc<OUT == OUT_X>(sub, lane, ring.acc[i][j], back);
            if constexpr (OUT == OUT_X) {
                sub.store<false>(ws + g.x + xm + ((int64_t)ci * g.sn + cj) * CELL, lane);
                sub.store<true>(ws + (op.to ? g.xt1 : g.xt0) + xm + ((int64_t)cj * g.sm + ci) * CELL, lane);
            } else {
                const int r0 = (g.trans ? cj : ci) * 32, c0 = (g.trans ? ci : cj) * 32;
                if (wide) {
#pragma unroll
                    for (int it = 0; it < 4; ++it) {
                        const int r = it * 8 + (lane >> 3), c = (lane & 7) * 4;
                        if (r0 + r >= rows || c0 + c >= cols) continue;
                        float o[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] = __builtin_bit_cast(float, g.trans ? sub.at[c + e][r] : sub.at[r][c + e]);
                        float4 w = old[j][it];
                        w.x = __builtin_fmaf(-rate, o[0], w.x * io.keep);
                        w.y = __builtin_fmaf(-rate, o[1], w.y * io.keep);
                        w.z = __builtin_fmaf(-rate, o[2], w.z * io.keep);
                        w.w = __builtin_fmaf(-rate, o[3], w.w * io.keep);
                        *reinterpret_cast<float4*>(param + (int64_t)(r0 + r) * cols + c0 + c) = w;
                    }
                    continue;
                }
#pragma unroll
                for (int it = 0; it < 16; ++it) {
                    const int r = it * 2 + (lane >> 5), c = lane & 31;
                    if (r0 + r >= rows || c0 + c >= cols) continue;
                    const float v = __builtin_bit_cast(float, g.trans ? sub.at[c][r] : sub.at[r][c]);
                    const float o = OUT == OUT_MUON ? v : v * rest;
                    if constexpr (OUT == OUT_MUON) {
                        float* w = param + (int64_t)(r0 + r) * cols + c0 + c;
                        *w = __builtin_fmaf(-rate, o, *w * io.keep);
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

// ---- matrices with a side of at most 32 --------------------------------------------------------------------------------------
// All of the iteration is a polynomial of S = G G^T applied to G, and S is 32 x 32: two passes over G (S; the product with
// the polynomial) instead of three per step, everything in fp64 on its matrix instructions, whose 16 digits the recursion
// S <- R S R, Q <- R Q (R = a + b S + c S S) cannot spend.  The norm is the trace of S.  A workgroup takes a part of the
// columns; where there is more than one, a first launch leaves the partial sums of S and a second one adds them, iterates (in
// every workgroup alike, 19 products of 32 x 32, each waiting for the one before) and applies.  Measured against the general path:
// 16 x 2048 35 us, there 118; 16 x 128 in one launch 24 us, there 75.
constexpr int TINY = 32, TINY_K = 128;
typedef double f64x4 __attribute__((ext_vector_type(4)));

// D = P Q of 32 x 32, Q symmetric: a wave has the 16 x 16 tile (wave / 2, wave % 2), row lane / 16 + 4 r, column lane % 16
__device__ __forceinline__ f64x4 tiny_product(const double (*p)[33], const double (*q)[33], int ti, int tj, int lane) {
    f64x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < 32; k += 4)
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64(p[16 * ti + (lane & 15)][k + (lane >> 4)], q[16 * tj + (lane & 15)][k + (lane >> 4)],
                                                   acc, 0, 0, 0);
    return acc;
}

enum { TINY_SUM, TINY_APPLY, TINY_BOTH };

template <typename T, bool MUON>
__global__ __launch_bounds__(256) void orth_tiny_kernel(Plan plan, Pointers ptr, Ends io, int what, int steps, double eps,
                                                        double* __restrict__ partial) {
    __shared__ float x[32][TINY_K + 4];
    __shared__ double s[32][33], q[32][33], r[32][33], m[32][33];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ti = wave >> 1, tj = wave & 1;
    int k = 0;
    while (k + 1 < plan.groups && (int)blockIdx.x >= plan.first_tile[k + 1]) ++k;
    const Group& g = plan.g[k];
    const int parts = plan.parts[k], in_group = blockIdx.x - plan.first_tile[k], idx = in_group / parts, part = in_group - idx * parts;
    const int mat = g.first + idx, cols = g.trans ? g.m : g.n;
    const int each = ((g.n + parts - 1) / parts + TINY_K - 1) / TINY_K * TINY_K;
    const int first = part * each, last = first + each < g.n ? first + each : g.n;
    const T* in = MUON ? nullptr : (const T*)io.in + mat * io.in_matrix;
    const float* gr = MUON ? ptr.grad[mat] : nullptr;
    float* mo = MUON ? ptr.momentum[mat] : nullptr;
    // columns c0 .. c0 + 127 of X (a row of the caller's matrix side by side in a wave); `update`: the momentum's step
    auto stage = [&](int c0, bool update) {
        __syncthreads();
        constexpr int EACH = 32 * TINY_K / 256;
        float v[EACH], gv[EACH];
#pragma unroll
        for (int l = 0; l < EACH; ++l) {                 // (all loads before the first use: their latency is paid once)
            const int e = threadIdx.x + 256 * l, i = g.trans ? e & 31 : e / TINY_K, c = g.trans ? e >> 5 : e % TINY_K;
            const bool in_range = i < g.m && c0 + c < last;
            const int row = in_range ? (g.trans ? c0 + c : i) : 0, col = in_range ? (g.trans ? i : c0 + c) : 0;
            if constexpr (MUON) {
                v[l] = mo[(int64_t)row * cols + col];
                gv[l] = gr[(int64_t)row * cols + col];
            } else {
                v[l] = (float)in[(int64_t)row * io.in_row + col];
            }
        }
#pragma unroll
        for (int l = 0; l < EACH; ++l) {
            const int e = threadIdx.x + 256 * l, i = g.trans ? e & 31 : e / TINY_K, c = g.trans ? e >> 5 : e % TINY_K;
            const bool in_range = i < g.m && c0 + c < last;
            if constexpr (MUON) {
                if (update) {
                    v[l] = __builtin_fmaf(io.momentum, v[l], gv[l]);
                    if (in_range) mo[(int64_t)(g.trans ? c0 + c : i) * cols + (g.trans ? i : c0 + c)] = v[l];
                }
                if (io.nesterov) v[l] = __builtin_fmaf(io.momentum, v[l], gv[l]);
            }
            x[i][c] = in_range ? v[l] : 0.f;
        }
        __syncthreads();
    };
    double* sums = partial + plan.partial[k] + (int64_t)idx * parts * (TINY * TINY);
    if (what != TINY_APPLY) {
        f64x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        for (int c0 = first; c0 < last; c0 += TINY_K) {
            stage(c0, true);
#pragma unroll 8
            for (int c = 0; c < TINY_K; c += 4)
                acc[c >> 2 & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)x[16 * ti + (lane & 15)][c + (lane >> 4)],
                                                                       (double)x[16 * tj + (lane & 15)][c + (lane >> 4)],
                                                                       acc[c >> 2 & 1], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 16 * ti + (lane >> 4) + 4 * e, col = 16 * tj + (lane & 15);
            if (what == TINY_SUM) sums[part * (TINY * TINY) + row * TINY + col] = acc[0][e] + acc[1][e];
            else s[row][col] = acc[0][e] + acc[1][e];
        }
        if (what == TINY_SUM) return;
    } else {
        for (int e = threadIdx.x; e < TINY * TINY; e += 256) {
            double v = 0;
            for (int p = 0; p < parts; ++p) v += sums[p * (TINY * TINY) + e];
            s[e >> 5][e & 31] = v;
        }
    }
    __syncthreads();
    double trace = 0;
    for (int i = 0; i < TINY; ++i) trace += s[i][i];
    const double scale = over_norm(sqrt(trace), eps);
    __syncthreads();
    for (int e = threadIdx.x; e < TINY * TINY; e += 256) {
        s[e >> 5][e & 31] = s[e >> 5][e & 31] * scale * scale;
        q[e >> 5][e & 31] = (e >> 5) == (e & 31);
    }
    __syncthreads();
    for (int step = 0; step < steps; ++step) {
        const f64x4 ss = tiny_product(s, s, ti, tj, lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 16 * ti + (lane >> 4) + 4 * e, col = 16 * tj + (lane & 15);
            r[row][col] = (row == col ? DA : 0.0) + DB * s[row][col] + DC * ss[e];
        }
        __syncthreads();
        const f64x4 rq = tiny_product(r, q, ti, tj, lane), rs = tiny_product(r, s, ti, tj, lane);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = 16 * ti + (lane >> 4) + 4 * e, col = 16 * tj + (lane & 15);
            q[row][col] = rq[e];
            m[row][col] = rs[e];
        }
        __syncthreads();
        if (step + 1 < steps) {
            const f64x4 sn = tiny_product(r, m, ti, tj, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[16 * ti + (lane >> 4) + 4 * e][16 * tj + (lane & 15)] = sn[e];
            __syncthreads();
        }
    }
    const float rate = MUON ? io.lr * sqrtf(fmaxf(1.f, g.trans ? (float)g.n / (float)g.m : (float)g.m / (float)g.n)) : 0.f;
    for (int c0 = first; c0 < last; c0 += TINY_K) {
        if (what == TINY_APPLY || last - first > TINY_K) stage(c0, false);
#pragma unroll
        for (int t = 0; t < 4; ++t) {                    // a wave's columns: 32 of the 128, both row tiles
            const int ri = t & 1, cj = wave * 2 + (t >> 1);
            f64x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < 32; c += 4)
                acc = __builtin_amdgcn_mfma_f64_16x16x4f64(q[16 * ri + (lane & 15)][c + (lane >> 4)],
                                                           (double)x[c + (lane >> 4)][16 * cj + (lane & 15)], acc, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 16 * ri + (lane >> 4) + 4 * e, j = c0 + 16 * cj + (lane & 15);
                if (i >= g.m || j >= last) continue;
                const float o = (float)(acc[e] * scale);
                const int row = g.trans ? j : i, col = g.trans ? i : j;
                if constexpr (MUON) {
                    float* w = ptr.param[mat] + (int64_t)row * cols + col;
                    *w = __builtin_fmaf(-rate, o, *w * io.keep);
                } else {
                    ((T*)io.out)[mat * io.out_matrix + (int64_t)row * io.out_row + col] = (T)o;
                }
            }
        }
    }
}

// ---- matrices that fit one workgroup's LDS ------------------------------------------------------------------------------------
// Sides of 33 to 96 whose X, X^T and S fit it (2 SM SN + SM SM cells of 4 KB; 64 x 256 and 96 x 128 at most): one launch for
// everything, a workgroup of eight waves per matrix with up to NC cells of X a wave.  The products are those of the general
// path, step by step.  Measured against it: 64 x 200 41 us, there 79; 96 x 128 41 us, there 83.
constexpr int SMALL_CELLS = 38;          // 152 KB

__device__ __forceinline__ f16x8 fragment(const char* cell, int h, int term, int lane) {
    return *reinterpret_cast<const f16x8*>(cell + (2 * h + term) * PIECE + lane * 16);
}

// acc += P Q^T of one cell pair's k block: the cross terms in an accumulator of their own (two chains instead of one)
__device__ __forceinline__ void terms(f32x16& acc, f32x16& cross, f16x8 a0, f16x8 a1, f16x8 b0, f16x8 b1) {
    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0, b1, cross, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a0, b0, acc, 0, 0, 0);
    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(a1, b0, cross, 0, 0, 0);
}

// acc += scale * (the cell whose transpose is `cell`): an accumulator's four rows are 8 bytes there
__device__ __forceinline__ void add_from(f32x16& acc, const char* cell, int lane, float scale) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const char* at = cell + (g >> 1) * 2 * PIECE + (g & 1) * 512 + (lane & 31) * 16 + (lane >> 5) * 8;
        const f16x4 hi = *reinterpret_cast<const f16x4*>(at), lo = *reinterpret_cast<const f16x4*>(at + PIECE);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[4 * g + e] = __builtin_fmaf(scale, (float)hi[e] + (float)lo[e], acc[4 * g + e]);
    }
}

// the sum over `cells` k cells of one cell's product
__device__ __forceinline__ f32x16 cell_product(const char* p, const char* q, int cells, int lane) {
    f32x16 acc, cross;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = cross[r] = 0.f;
#pragma unroll 2
    for (int k = 0; k < cells; ++k, p += CELL, q += CELL)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            terms(acc, cross, fragment(p, h, 0, lane), fragment(p, h, 1, lane), fragment(q, h, 0, lane), fragment(q, h, 1, lane));
    return acc + cross;
}

// scale * acc to its cell and to the transposed one.  A cell on the diagonal is its own transpose and is written once: of two
// entries that differ in their last bit, hi of one and lo of the other are a third value.
__device__ __forceinline__ void store_both(char* cell, char* transposed, const f32x16& acc, float scale, int lane) {
    char* mine = cell + ((lane >> 4) & 1) * 2 * PIECE + ((lane >> 3) & 1) * 512 + (lane & 7) * 2;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        f16x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            _Float16 h, l;
            split(scale * acc[4 * g + e], h, l);
            hi[e] = h;
            lo[e] = l;
            if (cell != transposed) {
                char* at = mine + (8 * g + 4 * (lane >> 5) + e) * 16;
                *reinterpret_cast<_Float16*>(at) = h;
                *reinterpret_cast<_Float16*>(at + PIECE) = l;
            }
        }
        char* at = transposed + (g >> 1) * 2 * PIECE + (g & 1) * 512 + (lane & 31) * 16 + (lane >> 5) * 8;
        *reinterpret_cast<f16x4*>(at) = hi;
        *reinterpret_cast<f16x4*>(at + PIECE) = lo;
    }
}

// The m x m side of a block of steps in one launch, for sides up to 128: a workgroup of eight waves per matrix, the operands of
// a product in two places of the LDS, every matrix's own values in fp32 registers (a wave has up to two cells i <= j of each).
// S comes as raw accumulators; T of alpha I + T goes to slot 0, scaled for MixOp.  A block of two steps has five products of 128 x 128, of
// three nine (27 us, against nine launches of 5 us and more): ten cells each on eight waves, so two waves have two of them while six wait.
template <int SM>
__global__ __launch_bounds__(512) void orth_chain_kernel(Plan plan, int block, int done, const double* __restrict__ norms,
                                                         const float* __restrict__ partial, char* __restrict__ ws) {
    constexpr int SYM = (SM * (SM + 1) / 2 + 7) / 8;
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int k = 0;
    while (k + 1 < plan.groups && (int)blockIdx.x >= plan.first_tile[k + 1]) ++k;
    const Group& g = plan.g[k];
    const int idx = blockIdx.x - plan.first_tile[k], parts = plan.parts[k], sm = g.sm;
    char *p = lds, *q = lds + SM * SM * CELL;
    int ci[SYM], cj[SYM];
#pragma unroll
    for (int u = 0; u < SYM; ++u) {
        int t = u * 8 + wave, i = 0;
        while (i < sm && t >= sm - i) t -= sm - i++;
        ci[u] = i;                                       // (sm: none)
        cj[u] = i + t;
    }
    struct Sym { f32x16 v[SYM]; };
    auto put = [&](char* to, const Sym& m, float scale) {
#pragma unroll
        for (int u = 0; u < SYM; ++u)
            if (ci[u] < sm) store_both(to + (ci[u] * SM + cj[u]) * CELL, to + (cj[u] * SM + ci[u]) * CELL, m.v[u], scale, lane);
    };
    // a A + b B + scale * (the product of what two places hold)
    auto mix = [&](const char* x, const char* y, float scale, float a, const Sym& ma, float b, const Sym& mb) {
        Sym r;
#pragma unroll
        for (int u = 0; u < SYM; ++u)
            if (ci[u] < sm) r.v[u] = a * ma.v[u] + (b * mb.v[u] + scale * cell_product(x + ci[u] * SM * CELL, y + cj[u] * SM * CELL, sm, lane));
        return r;
    };
    Sym s;
    const float to_s = ldexpf(1.f, -30 - 2 * raise_after(raise_in(norms, g.first + idx), done));
#pragma unroll
    for (int u = 0; u < SYM; ++u) {
        if (ci[u] >= sm) continue;
        const float* from = partial + plan.partial[k] + (int64_t)idx * parts * (16 * 1024) + (ci[u] * 4 + cj[u]) * 1024 + lane * 4;
#pragma unroll
        for (int r = 0; r < 16; ++r) s.v[u][r] = 0.f;
#pragma unroll 4
        for (int part = 0; part < parts; ++part, from += 16 * 1024)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 v = *reinterpret_cast<const float4*>(from + r * 256);
                s.v[u][4 * r] += v.x;
                s.v[u][4 * r + 1] += v.y;
                s.v[u][4 * r + 2] += v.z;
                s.v[u][4 * r + 3] += v.w;
            }
#pragma unroll
        for (int r = 0; r < 16; ++r) s.v[u][r] *= to_s;
    }
    put(p, s, 0x1p15f);
    __syncthreads();
    Sym t = mix(p, p, CC * 0x1p-30f, CB, s, 0.f, s);     // B = b S + c S S
    float scale = 0x1p14f;
    if (block > 1) {
        put(q, t, 0x1p14f);                              // q: B
        __syncthreads();
        Sym m = mix(q, p, 0x1p-29f, CA, s, 0.f, s);      // M = a S + B S
        __syncthreads();
        put(p, m, 0x1p15f);
        __syncthreads();
        s = mix(q, p, 0x1p-29f, CA, m, 0.f, m);          // S' = a M + B M
        __syncthreads();
        put(p, s, 0x1p15f);
        __syncthreads();
        Sym b = mix(p, p, CC * 0x1p-30f, CB, s, 0.f, s); // B'
        __syncthreads();
        put(p, b, 0x1p14f);
        __syncthreads();
        t = mix(p, q, 0x1p-28f, CA, t, CA, b);           // T' = a B + a B' + B' B
        scale = 0x1p11f;
        if (block > 2) {
            __syncthreads();
            put(q, s, 0x1p15f);
            __syncthreads();
            m = mix(p, q, 0x1p-29f, CA, s, 0.f, s);      // M'
            __syncthreads();
            put(q, m, 0x1p15f);
            __syncthreads();
            s = mix(p, q, 0x1p-29f, CA, m, 0.f, m);      // S''
            __syncthreads();
            put(q, s, 0x1p15f);
            __syncthreads();
            b = mix(q, q, CC * 0x1p-30f, CB, s, 0.f, s); // B''
            __syncthreads();
            put(q, b, 0x1p14f);
            put(p, t, 0x1p11f);
            __syncthreads();
            t = mix(q, p, 0x1p-25f, CA, t, CA * CA, b);  // T'' = a T' + a^2 B'' + B'' T'
            scale = 0x1p9f;
        }
    }
    char* out = ws + g.s + (int64_t)idx * sm * sm * CELL;
#pragma unroll
    for (int u = 0; u < SYM; ++u)
        if (ci[u] < sm) store_both(out + (ci[u] * sm + cj[u]) * CELL, out + (cj[u] * sm + ci[u]) * CELL, t.v[u], scale, lane);
}

template <int SM, int NC, typename T, bool MUON>
__global__ __launch_bounds__(512) void orth_small_kernel(Group g, Pointers ptr, Ends io, int steps, double eps) {
    constexpr int SYM = (SM * (SM + 1) / 2 + 7) / 8;     // cells i <= j of S a wave
    extern __shared__ __align__(16) char lds[];
    __shared__ double red[8];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cells = SM * g.sn, mat = g.first + blockIdx.x;
    char *x = lds, *xt = lds + cells * CELL, *s = lds + 2 * cells * CELL;
    const int rows = g.trans ? g.n : g.m, cols = g.trans ? g.m : g.n;
    const T* in = MUON ? nullptr : (const T*)io.in + mat * io.in_matrix;
    const float* gr = MUON ? ptr.grad[mat] : nullptr;
    float* mo = MUON ? ptr.momentum[mat] : nullptr;
    int raise;
    {
        float v[NC][16], gv[NC][16];
#pragma unroll
        for (int t = 0; t < NC; ++t) {
            const int c = t * 8 + wave, cj = c / SM, ci = c - cj * SM;
#pragma unroll
            for (int it = 0; it < 16; ++it) {
                const int r = (g.trans ? cj : ci) * 32 + it * 2 + (lane >> 5), col = (g.trans ? ci : cj) * 32 + (lane & 31);
                const bool in_range = c < cells && r < rows && col < cols;
                if constexpr (MUON) {
                    v[t][it] = in_range ? mo[(int64_t)r * cols + col] : 0.f;
                    gv[t][it] = in_range ? gr[(int64_t)r * cols + col] : 0.f;
                } else {
                    v[t][it] = in_range ? (float)in[(int64_t)r * io.in_row + col] : 0.f;
                }
            }
        }
        double sum = 0;
#pragma unroll
        for (int t = 0; t < NC; ++t)
#pragma unroll
            for (int it = 0; it < 16; ++it) {
                if constexpr (MUON) {
                    const int c = t * 8 + wave, cj = c / SM, ci = c - cj * SM;
                    const int r = (g.trans ? cj : ci) * 32 + it * 2 + (lane >> 5), col = (g.trans ? ci : cj) * 32 + (lane & 31);
                    v[t][it] = __builtin_fmaf(io.momentum, v[t][it], gv[t][it]);
                    if (c < cells && r < rows && col < cols) mo[(int64_t)r * cols + col] = v[t][it];
                    if (io.nesterov) v[t][it] = __builtin_fmaf(io.momentum, v[t][it], gv[t][it]);
                }
                sum += (double)v[t][it] * v[t][it];
            }
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) red[wave] = sum;
        __syncthreads();
        sum = 0;
        for (int w = 0; w < 8; ++w) sum += red[w];
        raise = raise_of(sqrt(sum), eps);
        const double scale = ldexp(over_norm(sqrt(sum), eps), raise + 15);
#pragma unroll
        for (int t = 0; t < NC; ++t) {
            const int c = t * 8 + wave, cj = c / SM, ci = c - cj * SM;
            if (c >= cells) continue;
#pragma unroll
            for (int it = 0; it < 16; ++it) {
                _Float16 hi, lo;
                split((float)((double)v[t][it] * scale), hi, lo);
                const int a = it * 2 + (lane >> 5), b = lane & 31, r = g.trans ? b : a, k = g.trans ? a : b;    // in X's cell
                char* to = x + (ci * g.sn + cj) * CELL + (k >> 4) * 2 * PIECE + (r + 32 * ((k >> 3) & 1)) * 16 + (k & 7) * 2;
                *reinterpret_cast<_Float16*>(to) = hi;
                *reinterpret_cast<_Float16*>(to + PIECE) = lo;
                to = xt + (cj * SM + ci) * CELL + (r >> 4) * 2 * PIECE + (k + 32 * ((r >> 3) & 1)) * 16 + (r & 7) * 2;
                *reinterpret_cast<_Float16*>(to) = hi;
                *reinterpret_cast<_Float16*>(to + PIECE) = lo;
            }
        }
    }
    __syncthreads();
    // the symmetric cells of this wave
    int si[SYM], sj[SYM];
#pragma unroll
    for (int u = 0; u < SYM; ++u) {
        int p = u * 8 + wave, i = 0;
        while (i < SM && p >= SM - i) p -= SM - i++;
        si[u] = i;                                       // (SM: none)
        sj[u] = i + p;
    }
    const float rate = MUON ? io.lr * sqrtf(fmaxf(1.f, (float)rows / (float)cols)) : 0.f;
    for (int step = 0; step < steps; ++step) {
        f32x16 sa[SYM], xa[NC];
        const int now = raise_after(raise, step), then = raise_after(raise, step + 1);
#pragma unroll
        for (int u = 0; u < SYM; ++u) {
            if (si[u] >= SM) continue;
            sa[u] = cell_product(x + si[u] * g.sn * CELL, x + sj[u] * g.sn * CELL, g.sn, lane);
            store_both(s + (si[u] * SM + sj[u]) * CELL, s + (sj[u] * SM + si[u]) * CELL, sa[u], ldexpf(1.f, -15 - 2 * now), lane);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < SYM; ++u) {
            if (si[u] >= SM) continue;
            sa[u] = cell_product(s + si[u] * SM * CELL, s + sj[u] * SM * CELL, SM, lane);
            add_from(sa[u], s + (sj[u] * SM + si[u]) * CELL, lane, CB / CC * 0x1p15f);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < SYM; ++u)
            if (si[u] < SM)
                store_both(s + (si[u] * SM + sj[u]) * CELL, s + (sj[u] * SM + si[u]) * CELL, sa[u], CC * 0x1p-16f, lane);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NC; ++t) {
            const int c = t * 8 + wave, cj = c / SM, ci = c - cj * SM;
            if (c >= cells) continue;
            xa[t] = cell_product(s + ci * SM * CELL, xt + cj * SM * CELL, SM, lane);
            add_from(xa[t], xt + (cj * SM + ci) * CELL, lane, CA * 0x1p14f);
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NC; ++t) {
            const int c = t * 8 + wave, cj = c / SM, ci = c - cj * SM;
            if (c >= cells) continue;
            if (step + 1 < steps) {
                store_both(x + (ci * g.sn + cj) * CELL, xt + (cj * SM + ci) * CELL, xa[t], ldexpf(1.f, -14 + then - now), lane);
                continue;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int i = ci * 32 + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), j = cj * 32 + (lane & 31);
                if (i >= g.m || j >= g.n) continue;
                const int r = g.trans ? j : i, col = g.trans ? i : j;
                const float o = ldexpf(xa[t][e], -29 - now);
                if constexpr (MUON) {
                    float* w = ptr.param[mat] + (int64_t)r * cols + col;
                    *w = __builtin_fmaf(-rate, o, *w * io.keep);
                } else {
                    ((T*)io.out)[mat * io.out_matrix + (int64_t)r * io.out_row + col] = (T)o;
                }
            }
        }
        __syncthreads();
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
inline int cells_of(int64_t n) { return (int)((n + 31) / 32); }

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

// first_tile of a launch with t x tj cells a workgroup; the number of tiles
int64_t count_tiles(Plan& plan, int t, int tj, bool sym) {
    int64_t total = 0;
    for (int k = 0; k < plan.groups; ++k) {
        const Group& g = plan.g[k];
        const int64_t ni = (g.sm + t - 1) / t, nj = (g.sn + tj - 1) / tj;
        plan.first_tile[k] = total > 0x7fffffff ? 0x7fffffff : (int)total;
        total += g.count * (sym ? ni * (ni + 1) / 2 : ni * nj);
    }
    plan.first_tile[plan.groups] = total > 0x7fffffff ? 0x7fffffff : (int)total;
    return total;
}

constexpr int CUS = 256;

// rows of cells of a workgroup in a launch of X's products
int cut_mix(Plan& plan, int64_t& tiles) {
    // 8 x 4 cells read each operand less often than 4 x 4: 4096 x 4096 4060 us instead of 4185, eight of 2048 x 2048 4000 and 4170,
    // the Muon step of two 4096 x 4096 and two 4096 x 2048 9226 and 9640.  But k loops below 64 cells do not carry their start
    // and end (256 of 256 x 512: 1125 us, with 4 x 4 1076; 64 of 512 x 512 level), and two of them fill a CU, so a round of 512
    // that is nearly empty costs more than that of smaller ones: three of 2100 x 2500, 540 tiles, 2190 and 2010 us; 612 tiles
    // 2435 and 2378, 640 level, 648 5345 and 5500.  Of a single round a quarter may be empty: 378 tiles 2565 and 2453, 390 2568
    // and 2676.
    int least = plan.g[0].sm;
    for (int k = 1; k < plan.groups; ++k) least = plan.g[k].sm < least ? plan.g[k].sm : least;
    tiles = count_tiles(plan, 8, 4, false);
    const int64_t places = (tiles + 2 * CUS - 1) / (2 * CUS) * (2 * CUS);
    if (least >= 64 && tiles * 8 >= places * (places > 2 * CUS ? 5 : 6)) return 8;
    // 4 x 4 cells against 2 x 2: k loops of up to 24 cells leave a large tile's start and end uncovered until several follow each
    // other on a CU (300 x 3000: eight 275 us with 2 x 2, 309 with 4 x 4; 32 of 380 x 4000 1576 and 1384); longer ones carry
    // them (1800 x 1800: 596 and 503 us)
    int most = 0;
    for (int k = 0; k < plan.groups; ++k) most = plan.g[k].sm > most ? plan.g[k].sm : most;
    if ((tiles = count_tiles(plan, 4, 4, false)) >= (most <= 24 ? 4 * CUS : CUS / 2)) return 4;
    tiles = count_tiles(plan, 2, 2, false);
    return 2;
}

// T of a launch of symmetric products; sets the plan's workgroups and parts, and the floats that the parts' accumulators
// take
int cut_sym(Plan& plan, bool from_x, bool raw, int64_t& workgroups, int64_t& floats) {
    floats = 0;
    int64_t work = 0, small_work = 0, most = 0;
    for (int k = 0; k < plan.groups; ++k) plan.parts[k] = 1;
    const int64_t tiles = count_tiles(plan, 4, 4, true);
    for (int k = 0; k < plan.groups; ++k) {
        const Group& g = plan.g[k];
        const int64_t n = (g.sm + 3) / 4, n2 = (g.sm + 1) / 2, cells = from_x ? g.sn : g.sm;
        work += g.count * (n * (n + 1) / 2) * cells;
        small_work += g.count * (n2 * (n2 + 1) / 2) * cells;
        most = cells > most ? cells : most;
    }
    // Small tiles where there are few large ones, or short k loops (up to 512) that leave a large tile's start and end uncovered:
    // small ones on the same CU overlap them.
    const bool large = tiles >= CUS / 2 && most > 16;
    // The k cells that a CU has to go through one after the other if all were equally busy, with two large workgroups on each or
    // a small one.  Parts pay for their second launch and a partial result's 64 KB out and in where the longest loop is 64
    // cells more than that (800 x 4096: 236 us with parts, 248 without; 16 of 300 x 3000: 475 and 399).  A part has a workgroup's
    // share, at least 16 cells; where that share fills the CUs, one workgroup more than fits would be another round
    // (2000 x 4000: 1008 us with three parts, 1082 with four).
    const int64_t even = large ? work / (2 * CUS) : small_work / CUS, share = work / (2 * CUS) > 16 ? work / (2 * CUS) : 16;
    workgroups = tiles;
    if (raw || most - even > 64) {
        workgroups = 0;
        for (int k = 0; k < plan.groups; ++k) {
            const Group& g = plan.g[k];
            const int64_t n = (g.sm + 3) / 4, cells = from_x ? g.sn : g.sm, count = g.count * (n * (n + 1) / 2);
            const int64_t parts = cells < share + share / 2 ? 1 : (raw || share == 16 ? cells + share - 1 : cells) / share;
            plan.parts[k] = (int)parts;
            plan.first_tile[k] = workgroups > 0x7fffffff ? 0x7fffffff : (int)workgroups;
            plan.partial[k] = floats;
            workgroups += count * parts;
            if (raw) floats += count * parts * 16 * 1024;
            else if (parts > 1) floats += 2 * count * parts * 16 * 1024;         // (two operations in a launch)
        }
        plan.first_tile[plan.groups] = workgroups > 0x7fffffff ? 0x7fffffff : (int)workgroups;
        return 4;
    }
    if (large) return 4;
    workgroups = count_tiles(plan, 2, 2, true);
    return 2;
}

// Steps can go through the m x m side in blocks: S after a step is R S R with R = a I + B, and j steps are one product of X
// with R .. R'.  A block of j steps takes (5 j - 4) m^3 instead of j m^3 flop in symmetric products and saves j - 1 passes
// over X, 3 m^2 n flop each.  The price is digits: the identity part alpha = a^j of the block's product cancels most of the
// largest singular values (their factor is near a^-j of it).  Frobenius errors measured against 64 bits, m >= 64, spectra
// from flat to four decades: 1.3e-6 to 5.9e-6 step by step (fp32 products: 1.3e-6 to 5.1e-6), at most 1.2 times that with
// two steps first, 2e-6 to 7.5e-6 with three and two.  So fp32 results and the Muon step (`exact`) get the first, 16-bit
// results, whose own rounding is 2e-4 and more, the second.  (The Muon step of five layers 784 -> 512 takes 1845 us; with three
// and two 1332, with three and single ones 1587, which on a spectrum of one strong direction over noise is 2 to 4 times
// further off than fp32 products.)  Below m = 64 (few rounding errors to average) and where X is not wide, step by step.
int next_block(const Plan& plan, bool exact, int done, int steps) {
    double wide = 0, square = 0;
    for (int k = 0; k < plan.groups; ++k) {
        const Group& g = plan.g[k];
        if (g.m < 64) return 1;
        wide += (double)g.count * g.m * g.m * g.n;
        square += (double)g.count * g.m * g.m * g.m;
    }
    if (wide < 1.25 * square) return 1;
    const int most = done == 0 ? (exact ? 2 : 3) : done == 3 && !exact ? 2 : 1, left = steps - done;
    return left < most ? left : most;
}

// The floats of cut_sym's parts do not grow with the count of matrices (more of them are cut into fewer parts), but a
// workspace for a count has to do for every smaller one.  This many do, for one group: t tiles of one matrix, at most `parts` a
// tile, and while a share is 16 cells (count t cells < 17 * 512) count t parts <= 17 * 512 parts / cells; larger shares make
// fewer parts, 512 * 18 / 17 and, where the last one of a tile may be short (raw), one a matrix more.
int64_t most_floats(const Plan& plan, bool from_x, bool raw) {
    const Group& g = plan.g[0];
    const int64_t n = (g.sm + 3) / 4, t = n * (n + 1) / 2, cells = from_x ? g.sn : g.sm;
    const int64_t parts = cells < 24 ? 1 : (cells + 15) / 16, all = g.count * t * parts;
    if (raw) return (all < 544 + g.count ? all : 544 + g.count) * 16 * 1024;
    // (whether there are any: the even share grows with the count but where tiles become large)
    const int64_t change = (CUS / 2 + t - 1) / t;
    bool any = false;
    for (const int64_t count : {(int64_t)1, change < g.count ? change : g.count}) {
        Plan some = plan;
        some.g[0].count = (int)count;
        int64_t workgroups, floats;
        cut_sym(some, from_x, false, workgroups, floats);
        any = any || floats;
    }
    const int64_t most = (17 * 512 - 1) * parts / cells;
    return any ? 2 * (all < most ? all : most) * 16 * 1024 : 0;
}

constexpr int SLOTS_CHAIN = 1, SLOTS_ONE = 2, SLOTS_TWO = 4, SLOTS_THREE = 5;

// Whether the m x m side is orth_chain_kernel's: all its matrices within 4 x 4 cells, and blocks of steps to save launches in
// (step by step it has one product, which two launches of 5 us do as fast).
bool chained(const Plan& plan, bool exact) {
    for (int k = 0; k < plan.groups; ++k)
        if (plan.g[k].sm > 4) return false;
    return next_block(plan, exact, 0, 3) > 1;
}

// the tiny groups' workgroups and parts; the doubles of their partial sums (0: one launch does it all)
int64_t cut_tiny(Plan& plan) {
    int64_t total = 0, doubles = 0;
    bool any = false;
    for (int k = 0; k < plan.groups; ++k) {
        const Group& g = plan.g[k];
        // (two rounds of one workgroup cost what a launch more does; past 64 parts adding them would)
        int64_t each = g.n <= 2 * TINY_K ? g.n : TINY_K;
        if ((g.n + each - 1) / each > 64) each = (g.n + 64 * TINY_K - 1) / (64 * TINY_K) * TINY_K;
        const int64_t parts = (g.n + each - 1) / each;
        plan.parts[k] = (int)parts;
        plan.partial[k] = doubles;
        plan.first_tile[k] = total > 0x7fffffff ? 0x7fffffff : (int)total;
        total += g.count * parts;
        any = any || parts > 1;
        doubles += g.count * parts * (TINY * TINY);
    }
    plan.first_tile[plan.groups] = total > 0x7fffffff ? 0x7fffffff : (int)total;
    return any ? doubles : 0;
}

// workspace: the tiny groups' partial sums (they are done with before the rest begins); over them the norms' and raises, the
// partial accumulators of split products, then each group's X, X^T (two) and slots (the small ones need none)
size_t layout(Plan& plan, Plan& tiny, bool exact, int64_t& partial) {
    const size_t doubles = (size_t)cut_tiny(tiny) * sizeof(double), least = doubles > 16 ? doubles : 16;
    if (!plan.groups) return least;
    const Group& end = plan.g[plan.groups - 1];
    const int matrices = end.first + end.count;
    int64_t at = (int64_t)matrices * NORM_STRIDE * sizeof(double);
    partial = at;
    int64_t most = 0;
    for (int from_x = 0; from_x < 2; ++from_x) {
        int64_t workgroups, floats;
        if (chained(plan, exact) && !from_x) continue;
        if (plan.groups == 1) floats = most_floats(plan, from_x, chained(plan, exact));
        else cut_sym(plan, from_x, chained(plan, exact), workgroups, floats);
        most = floats > most ? floats : most;
    }
    at += most * sizeof(float);
    const int block = next_block(plan, exact, 0, 3);
    const int slots = chained(plan, exact) ? SLOTS_CHAIN : block == 3 ? SLOTS_THREE : block == 2 ? SLOTS_TWO : SLOTS_ONE;
    for (int k = 0; k < plan.groups; ++k) {
        Group& g = plan.g[k];
        const int64_t x = (int64_t)g.count * g.sm * g.sn * CELL, s = (int64_t)g.count * g.sm * g.sm * CELL;
        g.x = at;
        g.xt0 = at + x;
        g.xt1 = at + 2 * x;
        g.s = at + 3 * x;
        at = g.s + slots * s;
    }
    return (size_t)at > least ? (size_t)at : least;
}

struct Job {
    Plan plan, small, tiny;              // the groups by the path they take
    Pointers ptr;
    Ends io;
    int steps;
    double eps;
    char* ws;
    int64_t partial;                     // offset of the partial accumulators
    hipStream_t stream;
};

template <int T, int RING>
int launch_sym(const Job& job, const SymOps& ops, int count, int64_t workgroups, bool parts, bool raw) {
    constexpr size_t lds = (size_t)RING * T * 4 * PIECE;
    static unsigned long long done;
    if (lds > 64 * 1024) {
        const int e = nf_raise_lds_cap((const void*)orth_sym_kernel<T, RING>, &done);
        if (e) return e;
    }
    float* partial = (float*)(job.ws + job.partial);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_sym_kernel<T, RING>), dim3((unsigned)workgroups, count), dim3(256), lds, job.stream,
                       job.plan, ops, (int)raw, (const double*)job.ws, partial, job.ws);
    const int e = nf_launch_status();
    if (e || !parts || raw) return e;
    if constexpr (T == 4) {
        Plan plan = job.plan;                            // the groups with parts, a wave a cell
        int64_t total = 0;
        int groups = 0;
        for (int k = 0; k < job.plan.groups; ++k) {
            if (job.plan.parts[k] == 1) continue;
            const Group& g = plan.g[groups] = job.plan.g[k];
            const int64_t n = (g.sm + 3) / 4;
            plan.parts[groups] = job.plan.parts[k];
            plan.partial[groups] = job.plan.partial[k];
            plan.first_tile[groups++] = (int)total;
            total += g.count * (n * (n + 1) / 2) * 4;
            if (total > 0x1fffffff) return NF_ERR_SHAPE;
        }
        plan.groups = groups;
        plan.first_tile[groups] = (int)total;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_sym_finish_kernel<T>), dim3((unsigned)total, count), dim3(256), 0, job.stream, plan,
                           ops, (const double*)job.ws, partial, job.ws);
        return nf_launch_status();
    }
    return NF_OK;
}

int sym(Job& job, const SymOps& ops, int count, bool raw = false) {
    int64_t workgroups, floats;
    const int t = cut_sym(job.plan, ops.op[0].p == FROM_X, raw, workgroups, floats);
    if (workgroups > 0x7fffffff) return NF_ERR_SHAPE;
    if (t == 4) return launch_sym<4, 4>(job, ops, count, workgroups, floats != 0, raw);
    return launch_sym<2, 6>(job, ops, count, workgroups, false, false);
}

template <int SM>
int launch_chain(const Job& job, const Plan& plan, int block, int done) {
    constexpr int lds = 2 * SM * SM * CELL;
    if (lds > 64 * 1024) {
        static unsigned long long done;
        const int e = nf_raise_lds_cap((const void*)orth_chain_kernel<SM>, &done);
        if (e) return e;
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_chain_kernel<SM>), dim3((unsigned)plan.first_tile[plan.groups]), dim3(512), lds, job.stream,
                       plan, block, done, (const double*)job.ws, (const float*)(job.ws + job.partial), job.ws);
    return nf_launch_status();
}

int chain(Job& job, int block, int done) {
    const SymOp op = {FROM_X, FROM_X, 0, NONE, NONE, 1.f, 0.f, 0.f};
    int e = sym(job, SymOps{{op, op}, done}, 1, true);
    if (e) return e;
    Plan plan = job.plan;                                // a workgroup a matrix
    int64_t total = 0;
    int most = 0;
    for (int k = 0; k < plan.groups; ++k) {
        plan.first_tile[k] = (int)total;
        total += plan.g[k].count;
        most = plan.g[k].sm > most ? plan.g[k].sm : most;
    }
    plan.first_tile[plan.groups] = (int)total;
    return most <= 2 ? launch_chain<2>(job, plan, block, done) : launch_chain<4>(job, plan, block, done);
}

int sym_one(Job& job, SymOp op, int done = 0) { return sym(job, SymOps{{op, op}, done}, 1); }

template <int TI, int TJ, int RING, int OUT>
int launch_mix(const Job& job, const MixOp& op, int64_t tiles) {
    constexpr size_t lds = (size_t)RING * (TI + TJ) * 2 * PIECE;
    static unsigned long long done;
    if (lds > 64 * 1024) {
        const int e = nf_raise_lds_cap((const void*)orth_mix_kernel<TI, TJ, RING, OUT>, &done);
        if (e) return e;
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_mix_kernel<TI, TJ, RING, OUT>), dim3((unsigned)tiles), dim3(256), lds, job.stream, job.plan,
                       job.ptr, job.io, op, (const double*)job.ws, job.ws);
    return nf_launch_status();
}

template <int OUT>
int mix(Job& job, const MixOp& op) {
    int64_t tiles;
    const int t = cut_mix(job.plan, tiles);
    if (tiles > 0x7fffffff) return NF_ERR_SHAPE;
    if (t == 8) return launch_mix<8, 4, 3, OUT>(job, op, tiles);
    if (t == 4) return launch_mix<4, 4, 4, OUT>(job, op, tiles);
    return launch_mix<2, 2, 6, OUT>(job, op, tiles);
}

// Scales (powers of two) of the slots: S and M = R S 15 (|M| < 1.45), B = b S + c S S 14, and of alpha I + T, the product of
// j steps' R, its T: 14 for one step (T = B), 11 for two (|T| <= a^2 = 11.9), 9 for three (40.9).
#define TWO(e) ldexpf(1.f, e)

template <typename T, bool MUON>
int run_tiny(const Job& job) {
    const Plan& plan = job.tiny;
    bool parts = false;
    for (int k = 0; k < plan.groups; ++k) parts = parts || plan.parts[k] > 1;
    for (int what = parts ? TINY_SUM : TINY_BOTH; what <= (parts ? TINY_APPLY : TINY_BOTH); ++what) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_tiny_kernel<T, MUON>), dim3((unsigned)plan.first_tile[plan.groups]), dim3(256), 0,
                           job.stream, plan, job.ptr, job.io, what, job.steps, job.eps, (double*)job.ws);
        const int e = nf_launch_status();
        if (e) return e;
    }
    return NF_OK;
}

// (nf_raise_lds_cap leaves no room for this kernel's static LDS)
int raise_lds(const void* kernel, unsigned long long* done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return (int)e;
    const unsigned long long bit = (dev >= 0 && dev < 64) ? 1ull << dev : 0ull;
    if (bit && (__atomic_load_n(done, __ATOMIC_ACQUIRE) & bit)) return NF_OK;
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, SMALL_CELLS * CELL);
    if (e != hipSuccess) return (int)e;
    if (bit) __atomic_fetch_or(done, bit, __ATOMIC_RELEASE);
    return NF_OK;
}

template <int SM, int NC, typename T, bool MUON>
int launch_small(const Job& job, const Group& g) {
    static unsigned long long done;
    const int e = raise_lds((const void*)orth_small_kernel<SM, NC, T, MUON>, &done);
    if (e) return e;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_small_kernel<SM, NC, T, MUON>), dim3(g.count), dim3(512), SM * (2 * g.sn + SM) * CELL, job.stream, g,
                       job.ptr, job.io, job.steps, job.eps);
    return nf_launch_status();
}

template <typename T, bool MUON>
int run_small(const Job& job) {
    for (int k = 0; k < job.small.groups; ++k) {
        const Group& g = job.small.g[k];
        const int nc = (g.sm * g.sn + 7) / 8;
        int e = NF_ERR_SHAPE;
        if (g.sm == 2) e = nc == 1 ? launch_small<2, 1, T, MUON>(job, g) : launch_small<2, 2, T, MUON>(job, g);
        else if (g.sm == 3) e = launch_small<3, 2, T, MUON>(job, g);
        if (e) return e;
    }
    return NF_OK;
}

template <typename T, bool MUON, int OUT>
int run(Job& job) {
    Plan& plan = job.plan;
    if (job.small.groups) {
        const int e = run_small<T, MUON>(job);
        if (e) return e;
    }
    if (job.tiny.groups) {
        if (job.tiny.first_tile[job.tiny.groups] == 0x7fffffff) return NF_ERR_SHAPE;
        const int e = run_tiny<T, MUON>(job);
        if (e) return e;
    }
    if (!plan.groups) return NF_OK;
    const int matrices = plan.g[plan.groups - 1].first + plan.g[plan.groups - 1].count;
    double* partial = (double*)job.ws;
    int64_t most = 1;
    for (int k = 0; k < plan.groups; ++k) {
        const int64_t size = (int64_t)plan.g[k].m * plan.g[k].n;
        most = size > most ? size : most;
    }
    int64_t blocks = (most + 4095) / 4096;
    if (blocks > NORM_BLOCKS) blocks = NORM_BLOCKS;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_norm_kernel<T, MUON>), dim3((unsigned)blocks, (unsigned)matrices), dim3(NORM_THREADS), 0,
                       job.stream, plan, job.ptr, job.io, partial);
    int e = nf_launch_status();
    if (e) return e;
    int64_t total = 0;
    for (int k = 0; k < plan.groups; ++k) {
        plan.first_tile[k] = (int)total;
        total += (int64_t)plan.g[k].count * (((int64_t)plan.g[k].sm * plan.g[k].sn + 3) / 4);
        if (total > 0x7fffffff) return NF_ERR_SHAPE;
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(orth_start_kernel<T, MUON>), dim3((unsigned)total), dim3(256), 0, job.stream, plan, job.ptr,
                       job.io, partial, (int)blocks, job.eps, job.ws);
    if ((e = nf_launch_status())) return e;
    const float a2 = CA * CA;
    constexpr bool exact = OUT != OUT_BF16 && OUT != OUT_F16;
    for (int s = 0, to = 1; s < job.steps; to ^= 1) {
        const int block = next_block(plan, exact, s, job.steps);
        MixOp op;
        if (chained(plan, exact)) {
            if ((e = chain(job, block, s))) return e;
            op = block == 1 ? MixOp{0, to, CA * TWO(14), TWO(-14)}
                            : block == 2 ? MixOp{0, to, a2 * TWO(11), TWO(-11)} : MixOp{0, to, a2 * CA * TWO(9), TWO(-9)};
            op.done = s;
            op.after = s += block;
            if ((e = s < job.steps ? mix<OUT_X>(job, op) : mix<OUT>(job, op))) return e;
            continue;
        }
        if ((e = sym_one(job, {FROM_X, FROM_X, 0, NONE, NONE, TWO(-15), 0.f, 0.f}, s))) return e;         // S = X X^T
        if ((e = sym_one(job, {0, 0, 1, 0, NONE, CC * TWO(-16), CB / CC * TWO(15), 0.f}))) return e;            // B
        if (block == 1) {
            op = {1, to, CA * TWO(14), TWO(-14)};
        } else {
            if ((e = sym_one(job, {1, 0, 2, 0, NONE, TWO(-14), CA * TWO(14), 0.f}))) return e;                       // M = a S + B S
            if ((e = sym_one(job, {1, 2, 3, 2, NONE, TWO(-14), CA * TWO(14), 0.f}))) return e;                       // S' = a M + B M
            if ((e = sym_one(job, {3, 3, 0, 3, NONE, CC * TWO(-16), CB / CC * TWO(15), 0.f}))) return e;        // B'
            const SymOps two = {{{0, 1, 2, 1, 0, TWO(-17), CA * TWO(14), CA * TWO(14)},                // T' = a B + a B' + B' B
                                 {0, 3, 4, 3, NONE, TWO(-14), CA * TWO(14), 0.f}}, 0};                           // M' = a S' + B' S'
            if ((e = sym(job, two, block - 1))) return e;
            op = {2, to, a2 * TWO(11), TWO(-11)};
            if (block == 3) {
                if ((e = sym_one(job, {0, 4, 1, 4, NONE, TWO(-14), CA * TWO(14), 0.f}))) return e;                   // S'' = a M' + B' M'
                if ((e = sym_one(job, {1, 1, 3, 1, NONE, CC * TWO(-16), CB / CC * TWO(15), 0.f}))) return e;    // B''
                if ((e = sym_one(job, {3, 2, 0, 2, 3, TWO(-16), CA * TWO(14), a2 * TWO(11)}))) return e;   // T'' = a T' + a^2 B'' + B'' T'
                op = {0, to, a2 * CA * TWO(9), TWO(-9)};
            }
        }
        op.done = s;
        op.after = s += block;
        if ((e = s < job.steps ? mix<OUT_X>(job, op) : mix<OUT>(job, op))) return e;
    }
    return NF_OK;
}

constexpr int MAX_MATRIX_GRID = 65535;   // matrices of one call (a grid's y extent)
constexpr int MAX_SIDE = 1 << 20;

bool sizes_ok(int64_t count, int rows, int cols) {
    return count >= 0 && count <= MAX_MATRIX_GRID && rows >= 1 && cols >= 1 && rows <= MAX_SIDE && cols <= MAX_SIDE;
}

// 0: the general path, 1: one workgroup's LDS, 2: tiny
int path_of(const int* shape) {
    const int sm = cells_of(shape[0] < shape[1] ? shape[0] : shape[1]), sn = cells_of(shape[0] < shape[1] ? shape[1] : shape[0]);
    return sm == 1 ? 2 : sm <= 3 && sm * (2 * sn + sm) <= SMALL_CELLS ? 1 : 0;
}
Plan& plan_of(Job& job, int path) { return path == 0 ? job.plan : path == 1 ? job.small : job.tiny; }
int longer(const int* shape) { return shape[0] > shape[1] ? shape[0] : shape[1]; }

// The matrices from `from` on that one sequence of launches takes, grouped by shape: `order` lists them group by group.
// Returns how many.
int plan_muon(const int* rows, const int* cols, int from, int count, Job& job, int* order) {
    int taken = 0, shapes[MAX_GROUPS][2], groups = 0, of[MAX_MATRICES];
    int64_t bytes = 0;
    while (from + taken < count && taken < MAX_MATRICES) {
        const int r = rows[from + taken], c = cols[from + taken];
        const Group g = group_of(r, c, 1, 0);
        bytes += ((int64_t)3 * g.sm * g.sn + (int64_t)SLOTS_THREE * g.sm * g.sm) * CELL;      // (at least what layout gives it)
        if (taken && bytes > SEQUENCE_BYTES) break;
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
    // where the general path runs anyway, what it does for matrices of 64 and more rows costs no launch of their own
    int path[MAX_GROUPS];
    bool general = false;
    for (int k = 0; k < groups; ++k) general = (path[k] = path_of(shapes[k])) == 0 || general;
    for (int k = 0; k < groups; ++k)
        if (general && path[k] == 1 && shapes[k][0] >= 64 && shapes[k][1] >= 64) path[k] = 0;
    // by path; the widest first: their workgroups run longest
    int at = 0, rank[MAX_GROUPS];
    for (int k = 0; k < groups; ++k) {
        int j = k;
        for (; j > 0; --j) {
            const int o = rank[j - 1];
            if (path[k] != path[o] ? path[k] > path[o] : longer(shapes[k]) <= longer(shapes[o])) break;
            rank[j] = o;
        }
        rank[j] = k;
    }
    for (int k = 0; k < groups; ++k) {
        const int first = at, shape = rank[k];
        for (int i = 0; i < taken; ++i)
            if (of[i] == shape) order[at++] = from + i;
        Plan& to = plan_of(job, path[shape]);
        to.g[to.groups++] = group_of(shapes[shape][0], shapes[shape][1], at - first, first);
    }
    return taken;
}

void plan_one(Job& job, int64_t count, int rows, int cols) {
    const int shape[2] = {rows, cols};
    Plan& to = plan_of(job, path_of(shape));
    to.groups = 1;
    to.g[0] = group_of(rows, cols, (int)count, 0);
}

}  // namespace

extern "C" size_t nf_orthogonalize_workspace_bytes(int64_t count, int rows, int cols, int elem) {
    if (!nf_elem_size(elem) || !sizes_ok(count, rows, cols) || count == 0) return 0;
    Job job = {};
    plan_one(job, count, rows, cols);
    return layout(job.plan, job.tiny, elem == NF_ELEM_F32, job.partial);
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
    Job job = {};
    plan_one(job, count, rows, cols);
    if (workspace_bytes < layout(job.plan, job.tiny, elem == NF_ELEM_F32, job.partial)) return NF_ERR_SCRATCH;
    job.io.in = matrices;
    job.io.out = out;
    job.io.in_matrix = matrix_stride;
    job.io.in_row = row_stride;
    job.io.out_matrix = out_matrix_stride;
    job.io.out_row = out_row_stride;
    job.steps = steps;
    job.eps = eps;
    job.ws = (char*)workspace;
    job.stream = (hipStream_t)stream;
    if (elem == NF_ELEM_F32) return run<float, false, OUT_F32>(job);
    if (elem == NF_ELEM_BF16) return run<__bf16, false, OUT_BF16>(job);
    return run<_Float16, false, OUT_F16>(job);
}

extern "C" size_t nf_muon_workspace_bytes(const int* rows, const int* cols, int count) {
    if (!rows || !cols) return 0;
    size_t most = 0;
    int order[MAX_MATRICES];
    for (int at = 0; at < count;) {
        for (int i = at; i < count && i < at + MAX_MATRICES; ++i)
            if (!sizes_ok(1, rows[i], cols[i])) return 0;
        Job job = {};
        const int taken = plan_muon(rows, cols, at, count, job, order);
        const size_t need = layout(job.plan, job.tiny, true, job.partial);
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
        Job job = {};
        const int taken = plan_muon(rows, cols, at, count, job, order);
        layout(job.plan, job.tiny, true, job.partial);
        for (int i = 0; i < taken; ++i) {
            job.ptr.grad[i] = grads[order[i]];
            job.ptr.momentum[i] = momenta[order[i]];
            job.ptr.param[i] = params[order[i]];
        }
        job.io.momentum = (float)momentum;
        job.io.nesterov = nesterov;
        job.io.keep = (float)(1.0 - lr * weight_decay);
        job.io.lr = (float)lr;
        job.steps = steps;
        job.eps = eps;
        job.ws = (char*)workspace;
        job.stream = (hipStream_t)stream;
        const int e = run<float, true, OUT_MUON>(job);
        if (e) return e;
        at += taken;
    }
    return NF_OK;
}
