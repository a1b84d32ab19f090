// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step built on it.
//   X_0 = U / (|U|_F + eps);   X <- B X,  B = a + b A + c A^2,  A = X X^T      over the shorter side, `steps` times
//   orthogonalize: out = X.   muon step: M <- mu M + s G;  U = s G + mu M (Nesterov) or M;
//                             W <- (1 - lr wd) W - lr f X      (f: a factor by the matrix' shape)
// X is m x n with m <= n: a matrix taller than wide is read and written transposed.
//
// Bound: the matrix pipe — m^2 n (A, half of it by symmetry) + m^3 (A^2, half) + 2 m^2 n flop a step against 8 bytes an element
// in and out; small matrices: launch latency.
//
// Arithmetic.  The iteration multiplies what is small in X_0 by up to a^5 = 485, its rounding errors with it, so that products of
// operands rounded to 8 or 11 bits are off by percents where a gradient's rank is below m (64 rows a batch: 1.7e-2 with one fp16
// plane in every step).  Every operand is kept as TWO fp16 planes, hi = fp16(x), lo = fp16(x - hi), 22 bits together, and a
// product is hi hi + (hi lo + lo hi) on v_mfma_f32_32x32x16_f16 with fp32 accumulators: what fp32 products give (the dropped
// lo lo is 2^-22 of a term at most) at a third of the fp16 rate instead of a sixteenth.  fp16's range is no limit: X_0 is U times a power of
// two (exact: the factor that is left of 1 / (|U| + eps) is applied to the first step's results), and every later operand has
// a bound that follows from |X_0| and the coefficients (ns_bounds) and is scaled by a power of two to stay below 2^15.
//
// Layout.  All products are C[i][j] = sum_k P[i][k] Q[j][k] with k contiguous in both operands: A = X X^T from X stored by rows,
// A^2 from A (symmetric), B X from B and X stored by columns.  So X is kept in both layouts.  Planes lie in the order in which the
// matrix instruction reads them (plane_at): a product's operands go through LDS as they are, and an epilogue's lanes write 512 bytes
// in a row.  Both sizes are padded to multiples of 32 with zeros, which stay zeros in every product.
#include <math.h>

#include <algorithm>
#include <exception>
#include <type_traits>
#include <vector>

#include "dgg_internal.h"

namespace dgg {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) float lds_f32;
typedef __attribute__((address_space(3))) half8 lds_half8;

constexpr int kNsMats = 16;      // matrices (stacks of them) per launch
constexpr int kNsSteps = 16;
constexpr int kNsParts = 1024;   // partial sums of squares per matrix, at most
constexpr int kThreads = 256;

struct NsMat {
    const void* in;          // U (orthogonalize) or the gradient
    void* out;               // X (orthogonalize) or the parameters, updated in place
    float* mom;              // muon: M, updated in place
    long long in_stride, out_stride, mom_stride;   // elements from one matrix of a stack to the next
    int ld_in, ld_out, ld_mom;
    int rows, cols, batch;
    int m, n, mp, np;        // short and long side, padded
    int turned;              // rows > cols
    int parts;               // workgroups of the norm pass per matrix
    int splits, kblocks;     // A = X X^T: ranges of 32-k blocks, blocks per range
    float step;              // muon: lr f
    // workspace (bytes from its start, for the whole stack)
    size_t xr, xt, a, b, slab, part, scal;
};

// One step's coefficients and the bounds that follow from them (ns_bounds): |B| <= grow, |X| <= r and <= times |X_0|; the same of the next X
struct NsStep { float a, b, c, grow, r, times, r_next, times_next; };

// The powers of two of one matrix in one step: X = planes * sx, planes of A, B and the next X = value * sa, sb, sx_next
struct NsScale { float sx, sa, sb, sx_next; };

enum { kNorm, kSplit, kGram, kSum, kSquare, kApply, kPhases };

// first workgroup of each matrix in one of the launches (none: INT_MAX)
struct NsFirst { int at[kNsMats]; };

struct NsUpdate { float mu, gscale; int nesterov; };

struct NsArgs {
    NsMat mat[kNsMats];
    char* ws;
    NsUpdate update;
    float decay;             // lr wd
    int adjust;
    double lr, eps;
    int steps;
    NsStep step[kNsSteps];
};

static_assert(sizeof(NsArgs) <= 4096 && sizeof(NsArgs) % 8 == 0, "kernel arguments");

// the matrix a workgroup works on, and its number among the matrix' workgroups
__device__ __forceinline__ int find(const NsFirst& f, int block, int& local) {
    int d = 0, at = 0;
#pragma unroll
    for (int i = 1; i < kNsMats; ++i)
        if (block >= f.at[i]) {
            d = i;
            at = f.at[i];
        }
    local = block - at;
    return d;
}

// Workgroups go to the 8 dies in turn; work items that follow each other share operands: each die takes a run of them, so that
// they meet in its L2.  (A grid is a permutation of its items for any size.)
__device__ __forceinline__ int by_die() {
    const int n = (int)gridDim.x, q = n >> 3, r = n & 7, die = (int)blockIdx.x & 7;
    return die * q + min(die, r) + ((int)blockIdx.x >> 3);
}

// Fragment order: the planes of a matrix with rows of k are cut into blocks of 32 rows x 16 k, 2 KB each: hi, then lo; in a plane
// lane l of the matrix instruction finds its 8 k (16 bytes) at l * 16.  A row group's blocks follow each other along k.
__host__ __device__ __forceinline__ size_t plane_bytes(int r, int k) { return (size_t)r * k * 4; }
// byte offset of (row, k) in the hi plane; lo: 1024 further on
__device__ __forceinline__ size_t plane_at(int row, int k, int kp) {
    return ((size_t)(row >> 5) * (kp >> 4) + (k >> 4)) * 2048 + ((k >> 3) & 1) * 512 + (row & 31) * 16 + (k & 7) * 2;
}

// A pointer that was read from memory could point anywhere, to the compiler: as a pointer to global memory it is not accessed by flat
// instructions, which also wait for LDS.
template <typename T> using Global = T __attribute__((address_space(1)));

// sum of v over the workgroup's N threads, in a fixed order, for every thread
template <int N> __device__ __forceinline__ double block_sum(double v, double* sh /* N / 64 */) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < N / 64; ++i) s += sh[i];
    return s;
}

// u of the muon step from the gradient and the momentum AFTER its update
__device__ __forceinline__ float muon_u(const NsUpdate& a, float g, float m) { return a.nesterov ? fmaf(a.mu, m, a.gscale * g) : m; }

// W of the muon step.  What is taken off — lr f x and lr wd w — is added up before the one rounding against w: lr wd is often below the
// spacing of fp32 under 1 (5e-8 for the trainers' lr 1e-4 and wd 5e-4), where 1 - lr wd as a factor would be 1.7 times too much decay or
// none at all.  (An infinite parameter stays one.)
__device__ __forceinline__ float muon_w(float w, float x, float step, float decay) {
    return fabsf(w) < INFINITY ? w - fmaf(step, x, decay * w) : fmaf(-step, x, (1.f - decay) * w);
}

// ------------------------------------------------------------------------------------------------ norm
// sum of squares in 64 bits, one partial a workgroup (muon: M is updated on the way).  Rows without gaps are one long row.
template <typename T, bool MUON>
__global__ __launch_bounds__(kThreads) void ns_norm_kernel(NsArgs a, NsFirst first) {
    __shared__ double sh[kThreads / 64];
    // the launches that follow find the arguments in device memory: 3 KB through the kernel arguments of each would be copied
    // by the host and read back over the bus every time
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < (int)(sizeof(NsArgs) / 8); i += kThreads) ((Global<uint64_t>*)a.ws)[i] = ((const uint64_t*)&a)[i];
    int local;
    const NsMat& M = a.mat[find(first, (int)blockIdx.x, local)];
    const int bat = local / M.parts, part = local - bat * M.parts;
    const Global<T>* in = (const Global<T>*)M.in + (size_t)bat * M.in_stride;
    Global<float>* mom = MUON ? (Global<float>*)M.mom + (size_t)bat * M.mom_stride : nullptr;
    const bool flat = M.ld_in == M.cols && (!MUON || M.ld_mom == M.cols);
    const long long total = (long long)M.rows * M.cols;
    // a workgroup's share: a range of the long row, or whole rows
    const long long per = flat ? ((total + M.parts - 1) / M.parts + 63) / 64 * 64 : 0;
    const int row0 = flat ? 0 : part, rows = flat ? 1 : M.rows, drow = flat ? 1 : M.parts;
    const long long c0 = flat ? part * per : 0, c1 = flat ? (c0 + per < total ? c0 + per : total) : M.cols;
    const NsUpdate up = a.update;
    double s = 0.0;
    for (int r = row0; r < rows; r += drow) {
        const Global<T>* g = in + (long long)r * M.ld_in;
        Global<float>* mr = MUON ? mom + (long long)r * M.ld_mom : nullptr;
        for (long long c = c0 + threadIdx.x; c < c1; c += 8 * kThreads) {   // eight elements in flight
            float u[8], m[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const long long at = c + e * kThreads < c1 ? c + e * kThreads : c;   // (beyond the end: the first once more, not used)
                u[e] = (float)g[at];
                if (MUON) m[e] = mr[at];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (c + e * kThreads >= c1) break;
                if (MUON) {
                    m[e] = fmaf(up.mu, m[e], up.gscale * u[e]);
                    mr[c + e * kThreads] = m[e];
                    u[e] = muon_u(up, u[e], m[e]);
                }
                s = fma((double)u[e], (double)u[e], s);
            }
        }
    }
    s = block_sum<kThreads>(s, sh);
    if (threadIdx.x == 0) ((Global<double>*)(a.ws + M.part))[(size_t)bat * M.parts + part] = s;
}

// ------------------------------------------------------------------------------------------------ planes of X_0
// x, y as hi + lo, rounded to nearest.  hi is one value, behind the compiler's back: fused into the product that x came from, the
// conversion that is stored and the one that lo is taken from could round apart (a step of fp16 where they do).
__device__ __forceinline__ void split2(float x, float y, half2& hi, half2& lo) {
    hi = half2{(_Float16)x, (_Float16)y};
    asm("" : "+v"(hi));
    lo = half2{(_Float16)fmaf(-1.f, (float)hi.x, x), (_Float16)fmaf(-1.f, (float)hi.y, y)};
}
template <int N> struct Halves { half2 e[N / 2]; };
template <int N> __device__ __forceinline__ void store_planes(char* p, const float (&v)[N]) {
    Halves<N> hi, lo;
#pragma unroll
    for (int e = 0; e < N / 2; ++e) split2(v[2 * e], v[2 * e + 1], hi.e[e], lo.e[e]);
    typedef uint32_t Bits __attribute__((ext_vector_type(N / 2)));
    *(Bits*)p = __builtin_bit_cast(Bits, hi);
    *(Bits*)(p + 1024) = __builtin_bit_cast(Bits, lo);
}

// eight k of a row, at their place in the hi plane
__device__ __forceinline__ void store8(char* p, const float (&v)[8]) { store_planes<8>(p, v); }

// the power of two that brings `bound` into [2^14, 2^15)
__device__ __forceinline__ float below(float bound) { return ldexpf(1.f, 14 - ilogbf(bound)); }

// one step's powers of two, from every operand's bound: the one of the coefficients, or, for a norm far below eps, what |X_0| can
// have grown to (a thread a step: none waits for the one before)
__device__ __forceinline__ void scales(const NsArgs& a, double norm, int k0, int k, NsScale* o) {
    const NsStep S = a.step[k];
    float r0 = (float)(norm / (norm + a.eps));
    if (!(r0 > 0x1p-40f)) r0 = 0x1p-40f;
    const float r = fminf(S.r, S.times * r0);
    NsScale z;
    z.sx = k ? 1.f / below(r) : (float)(1.0 / ldexp(norm + a.eps, k0));
    z.sa = below(r * r);
    z.sb = below(S.grow);
    z.sx_next = below(fminf(S.r_next, S.times_next * r0));
    o[k] = z;
}

// 64 x 64 of X: U read along its rows, written by rows and by columns of X as planes of U * 2^k
template <typename T, bool MUON>
__global__ __launch_bounds__(kThreads) void ns_split_kernel(const NsArgs* args, NsFirst first) {
    const NsArgs& a = *args;
    char* const ws = (char*)args;   // (they lie at its start)
    __shared__ double sh[kThreads / 64];
    __shared__ float t[64][65];   // [i][j] of X
    int local;
    const NsMat M = a.mat[find(first, (int)blockIdx.x, local)];
    const int ti = (M.mp + 63) / 64, tj = (M.np + 63) / 64;
    const int bat = local / (ti * tj), tile = local - bat * ti * tj, i0 = tile / tj * 64, j0 = tile % tj * 64;
    const Global<T>* in = (const Global<T>*)M.in + (size_t)bat * M.in_stride;
    const Global<float>* mom = MUON ? (Global<float>*)M.mom + (size_t)bat * M.mom_stride : nullptr;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r0 = M.turned ? j0 : i0, c0 = M.turned ? i0 : j0;   // of U
    const NsUpdate up = a.update;   // (read before anything is written: the compiler could not tell that it stays)
    float u[16], m[16];   // all of the tile is in flight while the norm is summed
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int r = min(r0 + q * 4 + wave, M.rows - 1), c = min(c0 + lane, M.cols - 1);   // (beyond: not used)
        u[q] = (float)in[(long long)r * M.ld_in + c];
        if (MUON) m[q] = mom[(long long)r * M.ld_mom + c];
    }
    double s = 0.0;
    for (int p = threadIdx.x; p < M.parts; p += kThreads) s += ((const double*)(ws + M.part))[(size_t)bat * M.parts + p];
    const double norm = sqrt(block_sum<kThreads>(s, sh));
    // 2^k |U| in [2^14, 2^15): no element of the planes is larger.  A zero, infinite or NaN norm keeps k = 0.
    const int k = norm > 0.0 && norm < INFINITY ? 14 - ilogb(norm) : 0;
    if (tile == 0 && (int)threadIdx.x < a.steps) scales(a, norm, k, threadIdx.x, (NsScale*)(ws + M.scal) + (size_t)bat * kNsSteps);
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const bool in_u = r0 + q * 4 + wave < M.rows && c0 + lane < M.cols;
        const float v = in_u ? ldexpf(MUON ? muon_u(up, u[q], m[q]) : u[q], k) : 0.f;
        if (M.turned) t[lane][q * 4 + wave] = v;
        else t[q * 4 + wave][lane] = v;
    }
    __syncthreads();
    char* xr = ws + M.xr + (size_t)bat * plane_bytes(M.mp, M.np);
    char* xt = ws + M.xt + (size_t)bat * 2 * plane_bytes(M.np, M.mp);
    // 64 rows of 64 k: 8 k a thread, twice per layout
    for (int q = threadIdx.x; q < 512; q += kThreads) {
        const int row = q & 63, k8 = (q >> 6) * 8;
        float v[8], w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = t[row][k8 + e];
            w[e] = t[k8 + e][row];
        }
        if (i0 + row < M.mp && j0 + k8 < M.np) store8(xr + plane_at(i0 + row, j0 + k8, M.np), v);
        if (j0 + row < M.np && i0 + k8 < M.mp) store8(xt + plane_at(j0 + row, i0 + k8, M.mp), w);
    }
}

// ------------------------------------------------------------------------------------------------ product
// C[i][j] = sum_k P[i][k] Q[j][k]: a workgroup of 2 x 2 waves owns a tile of 64 F x 64 F of C, a wave F x F blocks of 32 x 32.  P, Q: row
// group 0 of planes in fragment order; row groups beyond the last are read as the last (their results are not stored).
// A stage is 32 k of both operands, 16 F KB, copied by LDS-DMA as it lies (a fragment is 1 KB in a row, lane by lane: no bank
// conflicts, no swizzle).  S stages, S - 1 of them in flight; the fragments of the next 16 k are read while the current ones are
// multiplied.  F = 1 is bound by LDS (1.3 KB read a matrix instruction and as much again written every third, 128 B a cycle),
// F = 2 by half of that.  hi hi and the two cross terms have accumulators of their own: the small ones are not rounded at the
// size of the large.
template <int F, int S>
struct Prod {
    static constexpr int kTile = 64 * F, kStage = 16384 * F, kLds = S * kStage, kPieces = 4 * F;   // pieces a wave and stage
    f32x16 hh[F][F], cross[F][F];
    struct Frags { half8 ph[F], pl[F], qh[F], ql[F]; };

    template <int N> __device__ static __forceinline__ void wait() {   // all but the newest N pieces have landed; everyone's
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
    }
    __device__ __forceinline__ void multiply(const Frags& x) {
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) cross[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.ph[i], x.ql[j], cross[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) hh[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.ph[i], x.qh[j], hh[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) cross[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.pl[i], x.qh[j], cross[i][j], 0, 0, 0);
    }

    __device__ __forceinline__ void run(const char* P, int prow, int prows, const char* Q, int qrow, int qrows, int kp, int kb0, int kb1) {
        extern __shared__ char smem[];
        const unsigned lds = (unsigned)(size_t)(lds_char*)smem;
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wi = wave >> 1, wj = wave & 1;
        // of every row group a wave fetches one piece: a plane of 16 k
        const char* src[4 * F];
#pragma unroll
        for (int g = 0; g < 4 * F; ++g) {
            const int at = g < 2 * F ? min(prow / 32 + g, prows / 32 - 1) : min(qrow / 32 + g - 2 * F, qrows / 32 - 1);
            src[g] = (g < 2 * F ? P : Q) + (size_t)at * kp * 128 + wave * 1024 + lane * 16;
        }
        const int n = kb1 - kb0;
        auto fetch = [&](int s) {
            const unsigned to = lds + wave * 1024 + (unsigned)(s % S) * kStage;
#pragma unroll
            for (int g = 0; g < 4 * F; ++g)
                __builtin_amdgcn_global_load_lds(reinterpret_cast<const float*>(src[g] + (size_t)(kb0 + s) * 4096),
                                                 (lds_f32*)(size_t)(to + g * 4096), 16, 0, 0);
        };
        const unsigned at_p = lds + lane * 16 + wi * F * 4096, at_q = lds + lane * 16 + (2 + wj) * F * 4096;
        auto read = [&](int s, int kk, Frags& x) {
            const unsigned o = (unsigned)(s % S) * kStage + kk * 2048;
#pragma unroll
            for (int i = 0; i < F; ++i) {
                x.ph[i] = *(lds_half8*)(size_t)(at_p + o + i * 4096);
                x.ql[i] = *(lds_half8*)(size_t)(at_q + o + i * 4096 + 1024);
                x.qh[i] = *(lds_half8*)(size_t)(at_q + o + i * 4096);
                x.pl[i] = *(lds_half8*)(size_t)(at_p + o + i * 4096 + 1024);
            }
        };
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) hh[i][j][e] = cross[i][j][e] = 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (s < n) fetch(s);
        if (n >= S) wait<(S - 1) * kPieces>();
        else wait<0>();
        Frags even, odd;
        read(0, 0, even);
        for (int s = 0; s < n; ++s) {
            read(s, 1, odd);
            multiply(even);
            if (s + 1 < n) {
                // stage s + 1 has landed, and everyone has read all of stage s (their reads have returned: lgkmcnt): its place is free
                if (s + S <= n) wait<(S - 2) * kPieces>();
                else wait<0>();
                if (s + S < n) fetch(s + S);
                read(s + 1, 0, even);
            }
            multiply(odd);
        }
        wait<0>();   // the LDS is free for the epilogue
    }

    // The lane's elements of block (f, g): four runs q of four consecutive i, (i0 + 32 f + 8 q + e, j0 + 32 g).
    __device__ static __forceinline__ int i0() { return ((threadIdx.x >> 7) & 1) * 32 * F + ((threadIdx.x >> 5) & 1) * 4; }
    __device__ static __forceinline__ int j0() { return ((threadIdx.x >> 6) & 1) * 32 * F + (threadIdx.x & 31); }
    __device__ __forceinline__ float value(int f, int g, int q, int e) const { return hh[f][g][4 * q + e] + cross[f][g][4 * q + e]; }

    // v[q][e] -> w[q][0..7] at row ti() + 32 f, columns tj() + 32 g + 16 q ..: a 32 x 32 block is turned in 4.5 KB of LDS of the wave's
    // own (pitch 36: 16-byte stores, and reads of 32 rows on 32 banks)
    __device__ static __forceinline__ int ti() { return ((threadIdx.x >> 7) & 1) * 32 * F + (threadIdx.x & 31); }
    __device__ static __forceinline__ int tj() { return ((threadIdx.x >> 6) & 1) * 32 * F + ((threadIdx.x >> 5) & 1) * 8; }
    __device__ static __forceinline__ void turn(const float (&v)[4][4], float (&w)[2][8]) {
        extern __shared__ char smem[];
        const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
        float* t = reinterpret_cast<float*>(smem) + (threadIdx.x >> 6) * (32 * 36);
#pragma unroll
        for (int q = 0; q < 4; ++q) *reinterpret_cast<float4*>(t + r * 36 + 8 * q + 4 * h) = make_float4(v[q][0], v[q][1], v[q][2], v[q][3]);
        __builtin_amdgcn_wave_barrier();   // (the wave's own LDS, in order: no workgroup barrier)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 8; ++e) w[q][e] = t[(16 * q + 8 * h + e) * 36 + r];
        __builtin_amdgcn_wave_barrier();
    }
};

// tile number -> (ti, tj) with ti <= tj, of a t x t grid, row by row
__device__ __forceinline__ void upper(int tile, int t, int& ti, int& tj) {
    ti = 0;
    while (tile >= t - ti) {
        tile -= t - ti;
        ++ti;
    }
    tj = ti + tile;
}

__device__ __forceinline__ NsScale scale_of(const char* ws, const NsMat& M, int bat, int k) {
    return ((const NsScale*)(ws + M.scal))[(size_t)bat * kNsSteps + k];
}

// four k of a row, at their place in the hi plane: written, and read as the values they stand for
__device__ __forceinline__ void store4(char* p, const float (&v)[4]) { store_planes<4>(p, v); }
__device__ __forceinline__ void load4(const char* p, float (&v)[4]) {
    const half4 hi = *(const half4*)p, lo = *(const half4*)(p + 1024);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)hi[e] + (float)lo[e];
}

// A = X X^T, tiles on and above the diagonal, a range of k each: fp32 slabs [split][mp][mp], or A where one range is all of k
template <int S>
__global__ __launch_bounds__(kThreads) void ns_gram_kernel(const NsArgs* args, NsFirst first, int k) {
    using Pr = Prod<1, S>;
    const NsArgs& a = *args;
    char* const ws = (char*)args;   // (they lie at its start)
    int local;
    const NsMat M = a.mat[find(first, by_die(), local)];
    const int t = (M.mp + Pr::kTile - 1) / Pr::kTile, tiles = t * (t + 1) / 2, per = tiles * M.splits;
    const int bat = local / per, rest = local - bat * per, split = rest / tiles;
    int ti, tj;
    upper(rest - split * tiles, t, ti, tj);
    const char* x = ws + M.xr + (size_t)bat * plane_bytes(M.mp, M.np);
    Pr p;
    p.run(x, ti * Pr::kTile, M.mp, x, tj * Pr::kTile, M.mp, M.np, split * M.kblocks, min((split + 1) * M.kblocks, M.np / 32));
    if (ti * Pr::kTile + p.i0() >= M.mp || tj * Pr::kTile + p.j0() >= M.mp) return;   // (the same for all of a wave: sizes are multiples of 32)
    if (M.splits == 1) {   // all of k: A itself, and its mirror image
        const NsScale z = scale_of(ws, M, bat, k);
        char* A = ws + M.a + (size_t)bat * plane_bytes(M.mp, M.mp);
        const int i0 = ti * Pr::kTile, j0 = tj * Pr::kTile;
        float v[4][4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[q][e] = p.value(0, 0, q, e) * z.sx * z.sx * z.sa;   // (in this order, as in ns_sum_kernel)
            store4(A + plane_at(j0 + p.j0(), i0 + p.i0(), M.mp) + (q >> 1) * 2048 + (q & 1) * 512, v[q]);
        }
        if (ti == tj) return;
        float w[2][8];
        p.turn(v, w);
#pragma unroll
        for (int q = 0; q < 2; ++q) store8(A + plane_at(i0 + p.ti(), j0 + p.tj() + 16 * q, M.mp), w[q]);
        return;
    }
    float* slab = (float*)(ws + M.slab) + ((size_t)bat * M.splits + split) * M.mp * M.mp +
                  (size_t)(ti * Pr::kTile + p.i0()) * M.mp + tj * Pr::kTile + p.j0();
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) slab[(size_t)(8 * q + e) * M.mp] = p.value(0, 0, q, e);
}

// sums the slabs in order: planes of A, both triangles; 32 x 32 elements a workgroup
__global__ __launch_bounds__(kThreads) void ns_sum_kernel(const NsArgs* args, NsFirst first, int k) {
    const NsArgs& a = *args;
    char* const ws = (char*)args;   // (they lie at its start)
    __shared__ float t[32][33];
    int local;
    const NsMat M = a.mat[find(first, by_die(), local)];
    const int n32 = M.mp / 32, tiles = n32 * (n32 + 1) / 2, bat = local / tiles;
    int ti, tj;
    upper(local - bat * tiles, n32, ti, tj);
    const NsScale z = scale_of(ws, M, bat, k);
    const size_t slab = (size_t)M.mp * M.mp;
    const int r0 = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * 4;
    const float* p = (const float*)(ws + M.slab) + (size_t)bat * M.splits * slab + (size_t)(ti * 32 + r0) * M.mp + tj * 32 + c0;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int sp = 0; sp < M.splits; ++sp) {
        const float4 w = *reinterpret_cast<const float4*>(p + sp * slab);
        v.x += w.x;
        v.y += w.y;
        v.z += w.z;
        v.w += w.w;
    }
    const float* pv = &v.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) t[r0][c0 + e] = pv[e] * z.sx * z.sx * z.sa;   // (in this order: sx * sx alone may be below fp32's range)
    __syncthreads();
    // 8 k of a row a thread: the block, then its mirror image
    const int r = threadIdx.x & 31, k8 = ((threadIdx.x >> 5) & 3) * 8, mirror = threadIdx.x >> 7;
    if (mirror && ti == tj) return;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = mirror || (ti == tj && k8 + e < r) ? t[k8 + e][r] : t[r][k8 + e];
    char* A = ws + M.a + (size_t)bat * plane_bytes(M.mp, M.mp);
    store8(A + plane_at((mirror ? tj : ti) * 32 + r, (mirror ? ti : tj) * 32 + k8, M.mp), w);
}

// B = a + b A + c A^2, tiles on and above the diagonal and their mirror images
template <int S>
__global__ __launch_bounds__(kThreads) void ns_square_kernel(const NsArgs* args, NsFirst first, int k) {
    using Pr = Prod<1, S>;
    const NsArgs& a = *args;
    char* const ws = (char*)args;   // (they lie at its start)
    int local;
    const NsMat M = a.mat[find(first, by_die(), local)];
    const int t = (M.mp + Pr::kTile - 1) / Pr::kTile, tiles = t * (t + 1) / 2, bat = local / tiles;
    int ti, tj;
    upper(local - bat * tiles, t, ti, tj);
    const char* A = ws + M.a + (size_t)bat * plane_bytes(M.mp, M.mp);
    char* B = ws + M.b + (size_t)bat * plane_bytes(M.mp, M.mp);
    Pr p;
    const int i0 = ti * Pr::kTile, j0 = tj * Pr::kTile, i = i0 + p.i0(), j = j0 + p.j0();
    const bool on = i < M.mp && j < M.mp;   // (the same for all of a wave)
    const size_t at = on ? plane_at(j, i, M.mp) : 0;   // row j, k = i: A and B are symmetric
    float v[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) load4(A + at + (q >> 1) * 2048 + (q & 1) * 512, v[q]);
    const NsScale z = scale_of(ws, M, bat, k);
    const float ratio = z.sb / z.sa, fa = a.step[k].a * z.sb, fb = a.step[k].b * ratio, fc = a.step[k].c * ratio / z.sa;
    p.run(A, i0, M.mp, A, j0, M.mp, M.mp, 0, M.mp / 32);
    if (!on) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[q][e] = fmaf(fc, p.value(0, 0, q, e), fmaf(fb, v[q][e], i + 8 * q + e == j ? fa : 0.f));
        store4(B + at + (q >> 1) * 2048 + (q & 1) * 512, v[q]);
    }
    if (ti == tj) return;
    float w[2][8];
    p.turn(v, w);
#pragma unroll
    for (int q = 0; q < 2; ++q) store8(B + plane_at(i0 + p.ti(), j0 + p.tj() + 16 * q, M.mp), w[q]);
}

// What the last step writes: X in a type of the caller's, or the parameters
struct ToMuon {};

// X <- B X: planes in both layouts (Out = void), or (last step) the result
template <int F, int S, typename Out>
__global__ __launch_bounds__(kThreads, 2) void ns_apply_kernel(const NsArgs* args, NsFirst first, int k) {
    using Pr = Prod<F, S>;
    const NsArgs& a = *args;
    char* const ws = (char*)args;   // (they lie at its start)
    int local;
    const NsMat M = a.mat[find(first, by_die(), local)];
    const int ti = (M.mp + Pr::kTile - 1) / Pr::kTile, tj = (M.np + Pr::kTile - 1) / Pr::kTile;
    const int bat = local / (ti * tj), tile = local - bat * ti * tj, i0 = tile % ti * Pr::kTile, j0 = tile / ti * Pr::kTile;
    const char* B = ws + M.b + (size_t)bat * plane_bytes(M.mp, M.mp);
    const size_t xtb = plane_bytes(M.np, M.mp);
    const int flip = k & 1;   // which half of xt holds X
    const char* xt = ws + M.xt + ((size_t)bat * 2 + flip) * xtb;
    char* xt_next = ws + M.xt + ((size_t)bat * 2 + (flip ^ 1)) * xtb;
    char* xr = ws + M.xr + (size_t)bat * plane_bytes(M.mp, M.np);
    const NsScale z = scale_of(ws, M, bat, k);
    constexpr bool last = !std::is_same<Out, void>::value;
    const float fb = z.sx / z.sb * (last ? 1.f : z.sx_next), step = M.step, decay = a.decay;
    Pr p;
    p.run(B, i0, M.mp, xt, j0, M.np, M.mp, 0, M.mp / 32);
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int g = 0; g < F; ++g) {
            const int i = i0 + p.i0() + 32 * f, j = j0 + p.j0() + 32 * g;
            if (i >= M.mp || j >= M.np) continue;   // (the same for all of a wave)
            float v[4][4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[q][e] = fb * p.value(f, g, q, e);
            if constexpr (!last) {
                char* o = xt_next + plane_at(j, i, M.mp);
#pragma unroll
                for (int q = 0; q < 4; ++q) store4(o + (q >> 1) * 2048 + (q & 1) * 512, v[q]);
                float w[2][8];
                p.turn(v, w);
                o = xr + plane_at(i0 + p.ti() + 32 * f, j0 + p.tj() + 32 * g, M.np);
#pragma unroll
                for (int q = 0; q < 2; ++q) store8(o + q * 2048, w[q]);
            } else {
                const long long di = M.turned ? 1 : M.ld_out;
                const long long at = (size_t)bat * M.out_stride + (M.turned ? (long long)j * M.ld_out + i : (long long)i * M.ld_out + j);
                if constexpr (std::is_same<Out, ToMuon>::value) {
                    Global<float>* W = (Global<float>*)M.out + at;
                    float w[4][4];
                    const int jn = min(j, M.n - 1) - j;   // (beyond the end: an element inside, not used)
                    const long long dj = M.turned ? (long long)jn * M.ld_out : jn;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[q][e] = W[(min(i + 8 * q + e, M.m - 1) - i) * di + dj];
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (i + 8 * q + e < M.m && j < M.n) W[(8 * q + e) * di] = muon_w(w[q][e], v[q][e], step, decay);
                } else {
                    Global<Out>* o = (Global<Out>*)M.out + at;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (i + 8 * q + e < M.m && j < M.n) o[(8 * q + e) * di] = (Out)v[q][e];
                }
            }
        }
}

// ------------------------------------------------------------------------------------------------ small matrices
// A matrix whose planes fit the LDS of one workgroup (short side <= 32 and long side <= 512, or 64 and 192): the whole step in one
// launch, 16 waves.  What bounds it is the chain of 5 barriers a step: 12 x 512 33 us, 32 x 300 31 (general route: 86 and more).
// The same planes in the same order and scales as there: A = X X^T in ranges of k that meet in LDS, A^2 and B X one 32 x 32 block a wave.
// A short side of a few rows has short sums, and the planes' 22 bits are what its error consists of (12 x 512: 1.0 to 1.5e-6 of |X|
// where fp32 products give 0.7 to 1.1e-6).  The matrix instructions are no bound here: lo lo is multiplied too, and B, whose error
// stays the same for all of X, has a third plane (together 0.4 to 0.9e-6).
constexpr int kSmallThreads = 1024, kPart = 32 * 36;

__host__ __device__ __forceinline__ int small_splits(int mp) { return mp == 32 ? 4 : 2; }
__host__ __device__ __forceinline__ int small_tiles(int mp) { return mp == 32 ? 1 : 3; }
int small_lds(int mp, int np) { return mp * np * 8 + mp * mp * 8 + small_tiles(mp) * small_splits(mp) * kPart * 4; }

struct SmallFrags { half8 ph, pl, qh, ql; };
__device__ __forceinline__ void small_read(const char* p, const char* q, SmallFrags& x) {
    x.ph = *(const half8*)p;
    x.ql = *(const half8*)(q + 1024);
    x.qh = *(const half8*)q;
    x.pl = *(const half8*)(p + 1024);
}
__device__ __forceinline__ void small_multiply(const SmallFrags& x, f32x16& hh, f32x16& cross) {
    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.ph, x.ql, cross, 0, 0, 0);
    hh = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.ph, x.qh, hh, 0, 0, 0);
    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.pl, x.qh, cross, 0, 0, 0);
    cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.pl, x.ql, cross, 0, 0, 0);
}
// where a third plane of its own (1 KB a block) holds what lies at `at` of the hi plane
__device__ __forceinline__ size_t third(size_t at) { return (at >> 11 << 10) | (at & 1023); }
__device__ __forceinline__ void zero(f32x16& hh, f32x16& cross) {
#pragma unroll
    for (int e = 0; e < 16; ++e) hh[e] = cross[e] = 0.f;
}

// The four pieces of a step, for a workgroup whose X (n columns of it) lies in LDS; p: this lane's place in a fragment.
// A = X X^T: tiles (0, 0), (0, 1), (1, 1), a range of k each, a wave each -> part[tile * splits + range][j][i], pitch 36
__device__ __forceinline__ void small_gram(const char* xr, int np, int tiles, int splits, float* part) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    if (wave >= tiles * splits) return;
    const int tile = wave / splits, ti = tile >> 1, tj = (tile + 1) >> 1, n = np / 16, per = ((n + splits - 1) / splits + 1) & ~1;
    const int b = (wave - tile * splits) * per, e = min(b + per, n);   // (an even number of 16 k)
    const char *p = xr + ti * n * 2048 + lane * 16, *q = xr + tj * n * 2048 + lane * 16;
    f32x16 hh, cross;
    zero(hh, cross);
    for (int x = b; x < e; x += 2) {
        SmallFrags f[2];
        small_read(p + x * 2048, q + x * 2048, f[0]);
        small_read(p + x * 2048 + 2048, q + x * 2048 + 2048, f[1]);
        small_multiply(f[0], hh, cross);
        small_multiply(f[1], hh, cross);
    }
    float* o = part + wave * kPart + r * 36 + 4 * h;
#pragma unroll
    for (int y = 0; y < 4; ++y)
        *(float4*)(o + 8 * y) = make_float4(hh[4 * y] + cross[4 * y], hh[4 * y + 1] + cross[4 * y + 1], hh[4 * y + 2] + cross[4 * y + 2],
                                            hh[4 * y + 3] + cross[4 * y + 3]);
}
// a thread's 8 elements of A (row aj, i8 .. of its tile), the ranges added up in order; threads below tiles * 128
__device__ __forceinline__ void small_sum(const float* part, int splits, float (&v)[8]) {
    const int tile = threadIdx.x >> 7, aj = threadIdx.x & 31, i8 = ((threadIdx.x >> 5) & 3) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (int sp = 0; sp < splits; ++sp) {
        const float* o = part + (tile * splits + sp) * kPart + aj * 36 + i8;
        const float4 lo = *(const float4*)o, hi = *(const float4*)(o + 4);
        v[0] += lo.x; v[1] += lo.y; v[2] += lo.z; v[3] += lo.w;
        v[4] += hi.x; v[5] += hi.y; v[6] += hi.z; v[7] += hi.w;
    }
}
// planes of A from them, both triangles
__device__ __forceinline__ void small_a(float (&v)[8], const NsScale& z, int mp, char* A) {
    const int tile = threadIdx.x >> 7, ti = tile >> 1, tj = (tile + 1) >> 1, aj = threadIdx.x & 31, i8 = ((threadIdx.x >> 5) & 3) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * z.sx * z.sx * z.sa;
    store8(A + plane_at(tj * 32 + aj, ti * 32 + i8, mp), v);
    if (ti == tj) return;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        half2 hi, lo;
        split2(v[e], v[e + 1], hi, lo);
        char* o = A + plane_at(ti * 32 + i8 + e, tj * 32 + aj, mp);
        *(_Float16*)o = hi.x;
        *(_Float16*)(o + 1024) = lo.x;
        *(_Float16*)(o + 16) = hi.y;   // (the next row)
        *(_Float16*)(o + 1040) = lo.y;
    }
}
// B = a + b A + c A^2 in three planes, a block a wave
__device__ __forceinline__ void small_square(const char* A, char* B, char* B3, const NsStep& S, const NsScale& z, int mp) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5, T = mp / 32;
    if (wave >= T * T) return;
    const int ti = wave / T, tj = wave - ti * T, n = mp / 16, bcol = tj * 32 + r;
    const float ratio = z.sb / z.sa, fa = S.a * z.sb, fb = S.b * ratio, fc = S.c * ratio / z.sa;
    f32x16 hh, cross;
    zero(hh, cross);
    for (int x = 0; x < n; x += 2) {
        SmallFrags f[2];
#pragma unroll
        for (int y = 0; y < 2; ++y)
            small_read(A + (ti * n + x + y) * 2048 + lane * 16, A + (tj * n + x + y) * 2048 + lane * 16, f[y]);
        small_multiply(f[0], hh, cross);
        small_multiply(f[1], hh, cross);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int row = ti * 32 + 8 * q + 4 * h;
        float v[4], two[4];
        load4(A + plane_at(bcol, row, mp), v);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(fc, hh[4 * q + e] + cross[4 * q + e], fmaf(fb, v[e], row + e == bcol ? fa : 0.f));
        const size_t to = plane_at(bcol, row, mp);
        store4(B + to, v);
        load4(B + to, two);   // (as stored; what is left is exact)
        *(half4*)(B3 + third(to)) = half4{(_Float16)(v[0] - two[0]), (_Float16)(v[1] - two[1]), (_Float16)(v[2] - two[2]),
                                          (_Float16)(v[3] - two[3])};
    }
}
// Block (bi, bj) of B X: a lane has a column's rows; ROWS: the same values with the operands exchanged, a lane has a row's columns, as X
// by rows is written.  (One after the other: the accumulators of both do not fit beside the rest.)
template <bool ROWS>
__device__ __forceinline__ void small_apply(const char* B, const char* B3, const char* xt, int bi, int bj, int mp, float f, float (&v)[4][4]) {
    const int lane = threadIdx.x & 63;
    f32x16 hh, cross;
    zero(hh, cross);
    for (int x = 0, n = mp / 16; x < n; x += 2) {
        SmallFrags g[2];
        half8 b3[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const char *b = B + (bi * n + x + y) * 2048 + lane * 16, *c = xt + (bj * n + x + y) * 2048 + lane * 16;
            if (ROWS) small_read(c, b, g[y]);
            else small_read(b, c, g[y]);
            b3[y] = *(const half8*)(B3 + (bi * n + x + y) * 1024 + lane * 16);
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            if (ROWS) cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(g[y].ph, b3[y], cross, 0, 0, 0);
            else cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(b3[y], g[y].qh, cross, 0, 0, 0);
            small_multiply(g[y], hh, cross);
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[q][e] = f * (hh[4 * q + e] + cross[4 * q + e]);
}

template <typename In, bool MUON>
__global__ __launch_bounds__(kSmallThreads) void ns_small_kernel(NsArgs a, NsFirst first) {
    extern __shared__ char smem[];
    __shared__ double sh[kSmallThreads / 64];
    __shared__ NsScale sc[kNsSteps];
    int bat;
    const NsMat& M = a.mat[find(first, (int)blockIdx.x, bat)];
    const int mp = M.mp, np = M.np, T = mp / 32, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    char* xr = smem;
    char* xt = xr + mp * np * 4;
    char* A = xt + mp * np * 4;
    char* B = A + mp * mp * 4;
    float* part = (float*)(B + mp * mp * 4);
    char* B3 = (char*)part;   // (the partial sums of A have been added up by then)
    const Global<In>* in = (const Global<In>*)M.in + (size_t)bat * M.in_stride;
    Global<float>* mom = MUON ? (Global<float>*)M.mom + (size_t)bat * M.mom_stride : nullptr;
    // U as it lies in memory, 16 elements a thread at most, through LDS (fp32 [mp][np + 4], in the place of X by columns and the start of A)
    float* stage = (float*)xt;
    const int total = M.rows * M.cols, pitch = np + 4, units = mp * np / 8;
    const NsUpdate up = a.update;
    const float per_col = 1.f / (float)M.cols;
    for (int e = threadIdx.x; e < mp * pitch / 4; e += kSmallThreads) ((float4*)stage)[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    float u[16], m[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        const int e = min((int)threadIdx.x + t * kSmallThreads, total - 1), r = (int)(((float)e + 0.5f) * per_col), c = e - r * M.cols;
        u[t] = (float)in[(long long)r * M.ld_in + c];   // (e below 2^14: the quotient's error stays below the half)
        if (MUON) m[t] = mom[(long long)r * M.ld_mom + c];
    }
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        const int e = (int)threadIdx.x + t * kSmallThreads, r = (int)(((float)e + 0.5f) * per_col), c = e - r * M.cols;
        if (e >= total) break;
        if (MUON) {
            m[t] = fmaf(up.mu, m[t], up.gscale * u[t]);
            mom[(long long)r * M.ld_mom + c] = m[t];
            u[t] = muon_u(up, u[t], m[t]);
        }
        s = fma((double)u[t], (double)u[t], s);
        stage[M.turned ? c * pitch + r : r * pitch + c] = u[t];
    }
    const double norm = sqrt(block_sum<kSmallThreads>(s, sh));
    const int k0 = norm > 0.0 && norm < INFINITY ? 14 - ilogb(norm) : 0;   // (as in ns_split_kernel)
    if ((int)threadIdx.x < a.steps) scales(a, norm, k0, threadIdx.x, sc);
    // 8 k of a row a thread, two rounds at most: X by rows, and by columns once everyone has read
    float v[2][8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int q = threadIdx.x + t * kSmallThreads, i = q & (mp - 1), j = q / mp * 8, groups = np / 32;
        if (q >= units) break;
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = ldexpf(stage[i * pitch + j + e], k0);
        store8(xr + plane_at(i, j, np), w);
        const int g = (q >> 5) / groups, i8 = g * 8, col = ((q >> 5) - g * groups) * 32 + (q & 31);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[t][e] = ldexpf(stage[(i8 + e) * pitch + col], k0);
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int q = threadIdx.x + t * kSmallThreads, groups = np / 32, g = (q >> 5) / groups;
        if (q < units) store8(xt + plane_at(((q >> 5) - g * groups) * 32 + (q & 31), g * 8, mp), v[t]);
    }
    __syncthreads();
    const int splits = small_splits(mp), tiles = small_tiles(mp), r = lane & 31, h = lane >> 5;
    // B X: the block of this wave; the lane's elements are (i + 8 q + e, j)
    const float step = M.step, decay = a.decay;
    const bool mine = wave < T * (np / 32);
    const int bj = wave / T, bi = wave - bj * T, i = bi * 32 + 4 * h, j = bj * 32 + r;
    const long long di = M.turned ? 1 : M.ld_out, at = M.turned ? (long long)j * M.ld_out + i : (long long)i * M.ld_out + j;
    Global<float>* W = (Global<float>*)M.out + (size_t)bat * M.out_stride;
    const auto one = [&](int k, auto is_last) {   // (the last step apart: its addresses take registers)
        constexpr bool last = decltype(is_last)::value;
        const NsScale z = sc[k];
        float v[4][4], x[4][4];   // x: X by rows, or (last step) the parameters
        if (MUON && last) {   // (on their way during the step)
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int ic = min(i + 8 * q + e, M.m - 1), jc = min(j, M.n - 1);   // (beyond: not used)
                    x[q][e] = W[M.turned ? (long long)jc * M.ld_out + ic : (long long)ic * M.ld_out + jc];
                }
        }
        small_gram(xr, np, tiles, splits, part);
        __syncthreads();
        if ((int)threadIdx.x < tiles * 128) {
            float s[8];
            small_sum(part, splits, s);
            small_a(s, z, mp, A);
        }
        __syncthreads();
        small_square(A, B, B3, a.step[k], z, mp);
        __syncthreads();
        const float f = z.sx / z.sb * (last ? 1.f : z.sx_next);
        if (mine) {
            small_apply<false>(B, B3, xt, bi, bj, mp, f, v);
            if (!last) small_apply<true>(B, B3, xt, bi, bj, mp, f, x);
        }
        __syncthreads();   // everyone has read X: its place takes the next
        if (mine)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (!last) {
                    store4(xt + plane_at(j, i + 8 * q, mp), v[q]);
                    store4(xr + plane_at(bi * 32 + r, bj * 32 + 8 * q + 4 * h, np), x[q]);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (i + 8 * q + e >= M.m || j >= M.n) continue;
                    if (MUON) W[at + (8 * q + e) * di] = muon_w(x[q][e], v[q][e], step, decay);
                    else ((Global<In>*)M.out)[(size_t)bat * M.out_stride + at + (8 * q + e) * di] = (In)v[q][e];
                }
            }
        __syncthreads();
    };
    for (int k = 0; k + 1 < a.steps; ++k) one(k, std::false_type());
    one(a.steps - 1, std::true_type());
}

// ------------------------------------------------------------------------------------------------ narrow matrices
// A short side of up to 64 rows and a long one that one workgroup cannot hold: a workgroup owns kNarrow / mp columns of X, and a step is
// ONE launch.  A workgroup adds up everyone's share of A = X X^T (4 KB a tile each), makes B from it — the same B in every workgroup —,
// multiplies its columns and leaves their share of the next A.  Shares alternate between two places (a launch reads one and writes
// the other), columns of X are read by their own workgroup alone.  What bounds it is the launches, steps + 1 of them, and the sum of the
// shares: 12 x 4608 53 us, 64 x 4108 87 (the general route: 91 and 99); 64 x 8192, 64 workgroups, would take 112.  With half as many
// columns again a workgroup, 12 x 4608 takes 66 us and 64 x 4108 85.
constexpr int kNarrow = 8192, kNarrowThreads = 512, kNarrowParts = 64;
__host__ __device__ __forceinline__ int narrow_splits(int mp) { return mp == 32 ? 8 : 2; }
int narrow_lds(int mp) { return kNarrow * 8 + mp * mp * 8 + small_tiles(mp) * narrow_splits(mp) * kPart * 4; }

// the power of two of a norm (as in ns_split_kernel)
__device__ __forceinline__ int power_of(double norm) { return norm > 0.0 && norm < INFINITY ? 14 - ilogb(norm) : 0; }

// this workgroup's share of A -> memory
__device__ __forceinline__ void narrow_share(const float* part, int mp, Global<float>* to) {
    if ((int)threadIdx.x >= small_tiles(mp) * 128) return;
    const int tile = threadIdx.x >> 7, aj = threadIdx.x & 31, i8 = ((threadIdx.x >> 5) & 3) * 8;
    float v[8];
    small_sum(part, narrow_splits(mp), v);
    Global<f32x4>* o = (Global<f32x4>*)(to + (tile * 32 + aj) * 32 + i8);
    o[0] = f32x4{v[0], v[1], v[2], v[3]};
    o[1] = f32x4{v[4], v[5], v[6], v[7]};
}

// everyone's shares of A, two elements of each of N tiles a thread -> part, as small_gram leaves one range (all loads of some shares
// are in flight)
template <int N> __device__ __forceinline__ void narrow_sum(const Global<float>* shares, const float* weight, int C, float* part) {
    const int e = threadIdx.x * 2;
    f32x2 v[N];
#pragma unroll
    for (int t = 0; t < N; ++t) v[t] = f32x2{0.f, 0.f};
#pragma unroll N == 1 ? 16 : 6
    for (int c = 0; c < C; ++c) {
        const float f = weight[c] * weight[c];
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const f32x2 o = *(const Global<f32x2>*)(shares + ((size_t)c * N + t) * 1024 + e);
            v[t].x = fmaf(f, o.x, v[t].x);
            v[t].y = fmaf(f, o.y, v[t].y);
        }
    }
#pragma unroll
    for (int t = 0; t < N; ++t) *(f32x2*)(part + t * kPart + (e >> 5) * 36 + (e & 31)) = v[t];
}

// The columns of U (muon: M is updated on the way) as planes of U * 2^k, k of THEIR norm, and their share of the first A
template <typename In, bool MUON>
__global__ __launch_bounds__(kNarrowThreads) void ns_narrow_first_kernel(NsArgs a, NsFirst first) {
    extern __shared__ char smem[];
    __shared__ double sh[kNarrowThreads / 64];
    if (blockIdx.x == 0)   // (for the launches that follow: ns_norm_kernel)
        for (int i = threadIdx.x; i < (int)(sizeof(NsArgs) / 8); i += kNarrowThreads) ((Global<uint64_t>*)a.ws)[i] = ((const uint64_t*)&a)[i];
    int local;
    const NsMat& M = a.mat[find(first, (int)blockIdx.x, local)];
    const int bat = local / M.parts, chunk = local - bat * M.parts, mp = M.mp, nc = kNarrow / mp, j0 = chunk * nc, wide = min(nc, M.n - j0);
    char* xr = smem;
    float* stage = (float*)(xr + kNarrow * 4);   // fp32 [mp][nc + 4]
    float* part = (float*)(xr + kNarrow * 8 + mp * mp * 8);
    const Global<In>* in = (const Global<In>*)M.in + (size_t)bat * M.in_stride;
    Global<float>* mom = MUON ? (Global<float>*)M.mom + (size_t)bat * M.mom_stride : nullptr;
    const int pitch = nc + 4, line = M.turned ? M.m : wide, total = M.m * wide;   // line: elements side by side in memory
    const NsUpdate up = a.update;
    const float per_line = 1.f / (float)line;
    for (int e = threadIdx.x; e < mp * pitch / 4; e += kNarrowThreads) ((float4*)stage)[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    float u[16], m[16];
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        const int e = min((int)threadIdx.x + t * kNarrowThreads, total - 1), y = (int)(((float)e + 0.5f) * per_line), x = e - y * line;
        const long long r = M.turned ? j0 + y : y, c = M.turned ? x : j0 + x;   // (e below 2^13: the quotient's error stays below the half)
        u[t] = (float)in[r * M.ld_in + c];
        if (MUON) m[t] = mom[r * M.ld_mom + c];
    }
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int t = 0; t < 16; ++t) {
        const int e = (int)threadIdx.x + t * kNarrowThreads, y = (int)(((float)e + 0.5f) * per_line), x = e - y * line;
        if (e >= total) break;
        if (MUON) {
            m[t] = fmaf(up.mu, m[t], up.gscale * u[t]);
            mom[(long long)(M.turned ? j0 + y : y) * M.ld_mom + (M.turned ? x : j0 + x)] = m[t];
            u[t] = muon_u(up, u[t], m[t]);
        }
        s = fma((double)u[t], (double)u[t], s);
        stage[M.turned ? x * pitch + y : y * pitch + x] = u[t];
    }
    s = block_sum<kNarrowThreads>(s, sh);
    if (threadIdx.x == 0) ((Global<double>*)(a.ws + M.part))[(size_t)bat * M.parts + chunk] = s;
    const int k = power_of(sqrt(s));
    char* xt = a.ws + M.xt + ((size_t)bat * M.parts + chunk) * kNarrow * 4;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int q = threadIdx.x + t * kNarrowThreads, i = q & (mp - 1), j = q / mp * 8, groups = nc / 32;
        float w[8], v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = ldexpf(stage[i * pitch + j + e], k);
        store8(xr + plane_at(i, j, nc), w);
        const int g = (q >> 5) / groups, i8 = g * 8, col = ((q >> 5) - g * groups) * 32 + (q & 31);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ldexpf(stage[(i8 + e) * pitch + col], k);
        store8(xt + plane_at(col, i8, mp), v);
    }
    __syncthreads();
    small_gram(xr, nc, small_tiles(mp), narrow_splits(mp), part);
    __syncthreads();
    narrow_share(part, mp, (Global<float>*)(a.ws + M.slab) + ((size_t)bat * M.parts + chunk) * small_tiles(mp) * 1024);
}

template <typename In, bool MUON>
__global__ __launch_bounds__(kNarrowThreads) void ns_narrow_kernel(const NsArgs* args, NsFirst first, int k) {
    extern __shared__ char smem[];
    __shared__ double sh[kNarrowThreads / 64];
    __shared__ NsScale sc[kNsSteps];
    __shared__ float weight[kNarrowParts];
    const NsArgs& a = *args;
    char* const ws = (char*)args;   // (they lie at its start)
    int local;
    const NsMat M = a.mat[find(first, (int)blockIdx.x, local)];
    const int C = M.parts, bat = local / C, chunk = local - bat * C, mp = M.mp, T = mp / 32, nc = kNarrow / mp, j0 = chunk * nc;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5, tiles = small_tiles(mp);
    char *xr = smem, *xt = xr + kNarrow * 4, *A = xt + kNarrow * 4, *B = A + mp * mp * 4;
    float* part = (float*)(B + mp * mp * 4);
    char* B3 = (char*)part;
    char* const xt_ws = ws + M.xt + ((size_t)bat * C + chunk) * kNarrow * 4;
    const size_t half = (size_t)M.batch * C * tiles * 1024;   // floats of one of the two places of the shares
    const Global<float>* shares = (const Global<float>*)(ws + M.slab) + (k & 1) * half + (size_t)bat * C * tiles * 1024;
    const bool last = k + 1 == a.steps;
    // X, and what the last step needs of the parameters, on their way
    f32x4 x[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = ((const Global<f32x4>*)xt_ws)[threadIdx.x + q * kNarrowThreads];
    const int bj = wave / T, bi = wave - bj * T, i = bi * 32 + 4 * h, j = j0 + bj * 32 + r;
    const long long di = M.turned ? 1 : M.ld_out, at = M.turned ? (long long)j * M.ld_out + i : (long long)i * M.ld_out + j;
    Global<float>* W = (Global<float>*)M.out + (size_t)bat * M.out_stride;
    const float step = M.step, decay = a.decay;
    float v[4][4], y[4][4];   // y: X by rows, or (last step) the parameters
    if (MUON && last) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int ic = min(i + 8 * q + e, M.m - 1), jc = min(j, M.n - 1);   // (beyond: not used)
                y[q][e] = W[M.turned ? (long long)jc * M.ld_out + ic : (long long)ic * M.ld_out + jc];
            }
    }
    double s = 0.0, mine = 0.0;
    if ((int)threadIdx.x < C) s = mine = ((const Global<double>*)(ws + M.part))[(size_t)bat * C + threadIdx.x];
    const double norm = sqrt(block_sum<kNarrowThreads>(s, sh));
    const int k0 = power_of(norm);
    // the first shares are in their columns' own powers of two (a share of nothing counts as nothing, whatever its power)
    if ((int)threadIdx.x < C) weight[threadIdx.x] = k ? 1.f : mine > 0.0 ? ldexpf(1.f, k0 - power_of(sqrt(mine))) : 0.f;
    if (threadIdx.x == 0) scales(a, norm, k0, k, sc);
#pragma unroll
    for (int q = 0; q < 4; ++q) ((f32x4*)xt)[threadIdx.x + q * kNarrowThreads] = x[q];
    __syncthreads();
    const NsScale z = sc[k];
    if (tiles == 1) narrow_sum<1>(shares, weight, C, part);
    else narrow_sum<3>(shares, weight, C, part);
    __syncthreads();
    if ((int)threadIdx.x < tiles * 128) {
        float s[8];
        small_sum(part, 1, s);
        small_a(s, z, mp, A);
    }
    __syncthreads();
    small_square(A, B, B3, a.step[k], z, mp);
    __syncthreads();
    const float f = z.sx / z.sb * (last ? 1.f : z.sx_next) * weight[chunk];
    small_apply<false>(B, B3, xt, bi, bj, mp, f, v);
    if (!last) small_apply<true>(B, B3, xt, bi, bj, mp, f, y);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (!last) {
            store4(xt_ws + plane_at(j - j0, i + 8 * q, mp), v[q]);
            store4(xr + plane_at(bi * 32 + r, bj * 32 + 8 * q + 4 * h, nc), y[q]);
            continue;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i + 8 * q + e >= M.m || j >= M.n) continue;
            if (MUON) W[at + (8 * q + e) * di] = muon_w(y[q][e], v[q][e], step, decay);
            else ((Global<In>*)M.out)[(size_t)bat * M.out_stride + at + (8 * q + e) * di] = (In)v[q][e];
        }
    }
    if (last) return;
    __syncthreads();
    small_gram(xr, nc, tiles, narrow_splits(mp), part);
    __syncthreads();
    narrow_share(part, mp, (Global<float>*)(ws + M.slab) + ((k + 1) & 1) * half + ((size_t)bat * C + chunk) * tiles * 1024);
}

// ------------------------------------------------------------------------------------------------ host side
// Bounds of every step's operands from the coefficients alone.  |X_0| <= 1 in the 2-norm; with r = |X| the singular values lie in
// [0, r], so |A| <= r^2, |B| <= max |a + b s^2 + c s^4|, |X'| <= max |a s + b s^3 + c s^5| over [0, r], and no element exceeds
// its matrix' norm.  1 % is added for the roundings.
bool ns_bounds(const double* coef, int steps, NsStep* out) {
    double r = 1.0, times = 1.0;
    for (int k = 0; k < steps; ++k) {
        const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
        // largest |g| and |s g| with g = a + b t + c t^2, t = s^2, over t in [0, r^2]: at its ends and where g' or (s g)' is 0
        double t[5] = {0.0, r * r, -b / (2.0 * c), -1.0, -1.0}, mx = 0.0, mg = 0.0;
        const double d = 9.0 * b * b - 20.0 * a * c;
        if (d >= 0.0) {   // 5 c t^2 + 3 b t + a = 0, both roots without cancellation
            const double q = -0.5 * (3.0 * b + copysign(sqrt(d), b));
            t[3] = q / (5.0 * c);
            t[4] = a / q;
        }
        for (double v : t)
            if (v >= 0.0 && v <= r * r) {   // (also leaves out infinities and NaN of c = 0)
                const double g = fabs(a + (b + c * v) * v);
                mg = fmax(mg, g);
                mx = fmax(mx, sqrt(v) * g);
            }
        mx *= 1.01;
        mg *= 1.01;
        if (!isfinite(a + b + c) || !(mx < 1e6) || !(mx > 1e-6) || !(mg < 1e6)) return false;
        const double most = fmin(times * mg, 1e30);
        out[k] = {(float)a, (float)b, (float)c, (float)mg, (float)r, (float)times, (float)mx, (float)most};
        r = mx;
        times = most;
    }
    return true;
}

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }
size_t up(size_t v) { return (v + 255) / 256 * 256; }

int ns_check(const dgg_matrix* mats, int count, const char* who) {
    if (!mats || count < 1) {
        set_error_text("%s: no matrices", who);
        return DGG_ERR_INVALID;
    }
    for (int i = 0; i < count; ++i) {
        const dgg_matrix& m = mats[i];
        const long long lo = m.rows < m.cols ? m.rows : m.cols, hi = m.rows < m.cols ? m.cols : m.rows;
        if (m.rows < 1 || m.cols < 1 || m.batch < 1 || lo > 16384 || hi > (1 << 20) || lo * hi * m.batch > (1ll << 32) ||
            m.batch > (1 << 20)) {
            set_error_text("%s: matrix %d: %d x %d x %lld; 1 .. 16384 on the short and 2^20 on the long side, 2^32 elements", who, i,
                           m.rows, m.cols, (long long)m.batch);
            return DGG_ERR_INVALID;
        }
    }
    return DGG_OK;
}

enum { kSmall, kNarrowRoute, kGeneral, kRoutes };

int ns_kind(const dgg_matrix& m) {
    const int lo = m.rows < m.cols ? m.rows : m.cols, hi = m.rows < m.cols ? m.cols : m.rows;
    if (lo <= 32 ? hi <= 512 : lo <= 64 && hi <= 192) return kSmall;
    return lo <= 64 && hi <= (lo <= 32 ? 16384 : 6144) ? kNarrowRoute : kGeneral;   // (64 and 48 workgroups)
}

// The route that each kind of a call's matrices takes: a route's launches work on up to 16 matrices, and those that another kind
// needs anyway are shared where they have the places (30 x 2000, 100 x 2000 and 100 x 30: 129 us where the last had a launch of
// its own, 98 together).
struct NsRoutes {
    int of[kRoutes];
    NsRoutes(const dgg_matrix* mats, int count) {
        int n[kRoutes] = {0, 0, 0};
        for (int i = 0; i < count; ++i) ++n[ns_kind(mats[i])];
        const auto free = [](int used) { return (kNsMats - used % kNsMats) % kNsMats; };
        for (int r = 0; r < kRoutes; ++r) of[r] = r;
        if (n[kSmall] <= free(n[kNarrowRoute])) of[kSmall] = kNarrowRoute;
        if (n[kSmall] + n[kNarrowRoute] <= free(n[kGeneral])) of[kSmall] = of[kNarrowRoute] = kGeneral;
    }
};

// What every route needs to know of one matrix.
void ns_fill(const dgg_matrix& in, const NsArgs& a, NsMat& M) {
    M.in = in.in; M.out = in.out; M.mom = in.momentum;
    M.in_stride = in.in_stride; M.out_stride = in.out_stride; M.mom_stride = in.momentum_stride;
    M.ld_in = in.ld_in; M.ld_out = in.ld_out; M.ld_mom = in.ld_momentum;
    M.rows = in.rows; M.cols = in.cols; M.batch = (int)in.batch;
    M.turned = in.rows > in.cols;
    M.m = M.turned ? in.cols : in.rows;
    M.n = M.turned ? in.rows : in.cols;
    M.mp = ceil_div(M.m, 32) * 32;
    M.np = ceil_div(M.n, 32) * 32;
    const double f = a.adjust == DGG_MUON_SPECTRAL ? sqrt(fmax(1.0, (double)in.rows / in.cols)) : 0.2 * sqrt((double)M.n);
    M.step = (float)(a.lr * f);
}

// Sizes, workspace places and first workgroups of up to kNsMats matrices.
struct NsPlan {
    int grid[kPhases];
    NsFirst first[kPhases];
    int f_apply;   // tiles of 64 f in B X
    size_t bytes;
};

void ns_plan(const dgg_matrix* const* mats, int count, NsArgs& a, NsPlan& P) {
    size_t at = up(sizeof(NsArgs));   // (its device copy)
    for (int k = 0; k < kPhases; ++k) {
        P.grid[k] = 0;
        for (int i = 0; i < kNsMats; ++i) P.first[k].at[i] = 0x7fffffff;
    }
    // B X in tiles of 128 x 128 where they give every CU one (a generator's hidden matrices, 436 tiles: 31.5 us a launch against 34.4
    // with tiles of 64 x 64), else of 64 x 64 (512 x 4620, 148 against 584 tiles: 16.8 against 19.4 us)
    long long wide = 0;
    for (int i = 0; i < count; ++i) wide += mats[i]->batch * ceil_div(mats[i]->rows, 128) * ceil_div(mats[i]->cols, 128);
    P.f_apply = wide >= 256 ? 2 : 1;
    for (int i = 0; i < count; ++i) {
        const dgg_matrix& in = *mats[i];
        NsMat& M = a.mat[i];
        ns_fill(in, a, M);
        M.parts = ceil_div((long long)M.m * M.n, kThreads * 16);
        if (M.parts > kNsParts) M.parts = kNsParts;
        const int t = ceil_div(M.mp, 64), tiles = t * (t + 1) / 2;
        // two workgroups a CU share the k of A = X X^T, 256 k or more each (192 .. 768 workgroups: 26.8, 21.8 (256), 19.6 (512), 19.0 us
        // for the generator's matrices, 10.8 .. 11.6 for 512 x 4620; 128 x 128 tiles: 18.9 and 11.6)
        int splits = ceil_div(512, (long long)tiles * M.batch);
        if (splits > M.np / 256) splits = M.np / 256;
        // one range of all k, and no launch that sums, for few k or where the tiles alone fill the chip (a call for 512 x 256: 108 -> 104 us,
        // for 24 of 257 x 771: 272 -> 252 us)
        if (splits < 1 || M.np <= 512 || (long long)tiles * M.batch >= 256) splits = 1;
        M.kblocks = ceil_div(M.np / 32, splits);
        M.splits = ceil_div(M.np / 32, M.kblocks);
        const size_t b = (size_t)M.batch;
        M.xr = at;   at = up(at + b * plane_bytes(M.mp, M.np));
        M.xt = at;   at = up(at + b * 2 * plane_bytes(M.np, M.mp));
        M.a = at;    at = up(at + b * plane_bytes(M.mp, M.mp));
        M.b = at;    at = up(at + b * plane_bytes(M.mp, M.mp));
        M.slab = at; at = up(at + (M.splits > 1 ? b * M.splits * M.mp * M.mp * 4 : 0));
        M.part = at; at = up(at + b * M.parts * 8);
        M.scal = at; at = up(at + b * kNsSteps * sizeof(NsScale));
        const int n32 = M.mp / 32;
        const int blocks[kPhases] = {M.parts, t * ceil_div(M.np, 64), tiles * M.splits, M.splits > 1 ? n32 * (n32 + 1) / 2 : 0, tiles,
                                       ceil_div(M.mp, 64 * P.f_apply) * ceil_div(M.np, 64 * P.f_apply)};
        for (int k = 0; k < kPhases; ++k) {
            P.first[k].at[i] = P.grid[k];
            P.grid[k] += blocks[k] * M.batch;
        }
    }
    P.bytes = at;
}

// The same of the narrow route; returns its workgroups
int ns_narrow_plan(const dgg_matrix* const* mats, int count, NsArgs& a, NsFirst& first, int& lds, size_t& bytes) {
    size_t at = up(sizeof(NsArgs));   // (its device copy)
    int grid = 0;
    lds = 0;
    for (int i = 0; i < kNsMats; ++i) first.at[i] = 0x7fffffff;
    for (int i = 0; i < count; ++i) {
        NsMat& M = a.mat[i];
        ns_fill(*mats[i], a, M);
        M.parts = ceil_div(M.n, kNarrow / M.mp);
        const size_t wgs = (size_t)M.batch * M.parts;
        M.xt = at;   at = up(at + wgs * kNarrow * 4);
        M.slab = at; at = up(at + wgs * 2 * small_tiles(M.mp) * 4096);
        M.part = at; at = up(at + wgs * 8);
        if (narrow_lds(M.mp) > lds) lds = narrow_lds(M.mp);
        first.at[i] = grid;
        grid += (int)wgs;
    }
    bytes = at;
    return grid;
}

// Threads of a launch: below 2^32 (from there on a grid may be cut short without an error).  A matrix needs at most a workgroup for each
// 64 x 64 of its elements in every launch; up to 1024 more where the general route shares A's k between workgroups (ns_plan: 512) and sums.
constexpr long long kNsMost = (1ll << 32) - 1024ll * kNsMats * kThreads - 1;
long long ns_threads(const dgg_matrix& m, int route) {
    const int lo = m.rows < m.cols ? m.rows : m.cols, hi = m.rows < m.cols ? m.cols : m.rows;
    if (route == kSmall) return (long long)m.batch * kSmallThreads;
    if (route == kNarrowRoute) return (long long)m.batch * ceil_div(hi, kNarrow / (lo <= 32 ? 32 : 64)) * kNarrowThreads;
    return (long long)m.batch * ceil_div(lo, 64) * ceil_div(hi, 64) * kThreads;
}

// up to kNsMats matrices of one route that a launch has the threads for, from mats[at] on; at moves behind them
int ns_group(const dgg_matrix* mats, int count, const NsRoutes& routes, int route, int& at, const dgg_matrix** group) {
    int n = 0;
    long long threads = 0;
    for (; at < count && n < kNsMats; ++at) {
        if (routes.of[ns_kind(mats[at])] != route) continue;
        threads += ns_threads(mats[at], route);
        if (n > 0 && threads > kNsMost) break;
        group[n++] = mats + at;
    }
    return n;
}

int64_t ns_need(const dgg_matrix* mats, int count, const char* who) {
    const dgg_matrix* group[kNsMats];
    size_t need = 256;
    const NsRoutes routes(mats, count);
    for (int i = 0; i < count; ++i)
        if (ns_threads(mats[i], routes.of[ns_kind(mats[i])]) > kNsMost) {
            set_error_text("%s: matrix %d: a stack of %lld of %d x %d needs a launch of 2^32 threads or more", who, i, (long long)mats[i].batch,
                           mats[i].rows, mats[i].cols);
            return DGG_ERR_INVALID;
        }
    for (int at = 0, n; (n = ns_group(mats, count, routes, kNarrowRoute, at, group)) > 0;) {
        NsArgs a = {};
        NsFirst first;
        size_t bytes;
        int lds;
        ns_narrow_plan(group, n, a, first, lds, bytes);
        if (bytes > need) need = bytes;
    }
    for (int at = 0, n; (n = ns_group(mats, count, routes, kGeneral, at, group)) > 0;) {
        NsArgs a = {};
        NsPlan P;
        ns_plan(group, n, a, P);
        if (P.bytes > need) need = P.bytes;
    }
    return (int64_t)need;
}

// What one matrix or stack covers in memory (bytes), for the check below: rows `row` wide and `ld` apart, matrices `one` long and `stride`
// apart.  A stack of single rows is one matrix.
struct NsSpan {
    uintptr_t lo, hi, ld, stride, row, one;
    int rows, batch;
    bool written;
};

// Every element of `a` lies in one of the places lo + k period + [0, length); do those of b, moved to them by multiples of the period,
// lie between two such places?
bool ns_between(const NsSpan& a, uintptr_t period, uintptr_t length, const NsSpan& b) {
    uintptr_t wide = b.hi - b.lo;   // what b covers once its own repetitions by multiples of the period are left out
    if (b.batch == 1 || b.stride % period == 0) wide = b.rows == 1 || b.ld % period == 0 ? b.row : b.one;
    const uintptr_t d = a.lo <= b.lo ? (b.lo - a.lo) % period : (period - (a.lo - b.lo) % period) % period;
    return d >= length && d + wide <= period;
}

// Two spans share no element: they lie one behind the other, or one lies in the gaps between the rows or the matrices of the other
// (column blocks of one wider buffer, stacks that alternate).
bool ns_free(const NsSpan& a, const NsSpan& b) {
    if (a.hi <= b.lo || b.hi <= a.lo) return true;
    const auto gaps = [](const NsSpan& p, const NsSpan& q) {
        return (p.rows > 1 && (p.batch == 1 || p.stride % p.ld == 0) && ns_between(p, p.ld, p.row, q)) ||
               (p.batch > 1 && p.stride > 0 && ns_between(p, p.stride, p.one, q));
    };
    return gaps(a, b) || gaps(b, a);
}

// What a call writes is written once and read by nothing else in it, only an output may be its own matrix' input: launches read an
// operand more than once and in no order between matrices.
bool ns_disjoint(const dgg_matrix* mats, int count, size_t size, bool muon) {
    std::vector<NsSpan> spans;
    spans.reserve((size_t)count * 3);
    for (int i = 0; i < count; ++i) {
        const dgg_matrix& m = mats[i];
        const auto put = [&](const void* p, int64_t ld, int64_t stride, bool written) {
            const uintptr_t lo = (uintptr_t)p, row = (uintptr_t)m.cols * size, one = (uintptr_t)(m.rows - 1) * ld * size + row;
            if (written && m.batch > 1) {   // the matrices of a stack: one behind the other, or side by side
                const bool behind = (uintptr_t)stride * size >= one;
                const bool beside = stride >= m.cols && (uintptr_t)(m.batch - 1) * stride * size + row <= (uintptr_t)ld * size;
                if (!behind && !beside) return false;
            }
            const uintptr_t hi = lo + (uintptr_t)(m.batch - 1) * stride * size + one, pitch = (uintptr_t)(m.rows > 1 ? ld : stride) * size;
            if (m.rows > 1) spans.push_back({lo, hi, pitch, (uintptr_t)stride * size, row, one, m.rows, (int)m.batch, written});
            else spans.push_back({lo, hi, pitch, 0, row, hi - lo, pitch ? (int)m.batch : 1, 1, written});
            return true;
        };
        const bool same = !muon && m.in == m.out && m.ld_in == m.ld_out && (m.batch == 1 || m.in_stride == m.out_stride);
        if (!put(m.out, m.ld_out, m.out_stride, true)) return false;
        if (!same && !put(m.in, m.ld_in, m.in_stride, false)) return false;
        if (muon && !put(m.momentum, m.ld_momentum, m.momentum_stride, true)) return false;
    }
    std::sort(spans.begin(), spans.end(), [](const NsSpan& a, const NsSpan& b) { return a.lo < b.lo; });
    for (size_t i = 0; i < spans.size(); ++i)
        for (size_t j = i + 1; j < spans.size() && spans[j].lo < spans[i].hi; ++j)
            if ((spans[i].written || spans[j].written) && !ns_free(spans[i], spans[j])) return false;
    return true;
}

// More than 64 KB of LDS has to be asked for, on every device that launches: always the most a kernel may need, so that another
// thread's call does not lower it in between.
bool ns_lds(const void* kernel, int bytes, const char* who) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) set_error(who, e);
    return e == hipSuccess;
}

template <typename T, bool MUON>
int ns_run(const dgg_matrix* mats, int count, NsArgs& a, const double* coef, int steps, void* ws, size_t ws_bytes,
           hipStream_t st, const char* who) {
    if (steps < 1 || steps > kNsSteps || !coef || !(a.eps >= 0.0) || !ns_bounds(coef, steps, a.step)) {
        set_error_text("%s: 1 .. %d steps, eps >= 0 and coefficients whose iterates stay bounded (|X| < 1e6) are needed", who, kNsSteps);
        return DGG_ERR_INVALID;
    }
    for (int i = 0; i < count; ++i) {
        const dgg_matrix& m = mats[i];
        const bool mom = !MUON || (m.momentum && m.ld_momentum >= m.cols && m.momentum_stride >= 0);
        if (!m.in || !m.out || !mom || m.ld_in < m.cols || m.ld_out < m.cols || m.in_stride < 0 || m.out_stride < 0) {
            set_error_text("%s: matrix %d: null pointer, a pitch below %d columns or a negative stride", who, i, m.cols);
            return DGG_ERR_INVALID;
        }
    }
    if (!ws || (uintptr_t)ws % 256) {
        set_error_text("%s: a 256-byte aligned workspace is needed", who);
        return DGG_ERR_WORKSPACE;
    }
    a.ws = (char*)ws;
    a.steps = steps;
    NsPlan P;
    const dgg_matrix* group[kNsMats];
    const int64_t need = ns_need(mats, count, who);
    if (need < 0) return (int)need;
    if ((int64_t)ws_bytes < need) {
        set_error_text("%s: the workspace has %zu bytes, %lld are needed", who, ws_bytes, (long long)need);
        return DGG_ERR_WORKSPACE;
    }
    bool disjoint = false;
    try {
        disjoint = ns_disjoint(mats, count, sizeof(T), MUON);
    } catch (const std::exception& e) {
        set_error_text("%s: %s", who, e.what());
        return DGG_ERR_INVALID;
    }
    if (!disjoint) {
        set_error_text("%s: what is written overlaps itself or another operand", who);
        return DGG_ERR_INVALID;
    }
    const NsRoutes routes(mats, count);
    for (int at = 0, n; (n = ns_group(mats, count, routes, kSmall, at, group)) > 0;) {
        NsFirst first;
        int grid = 0, lds = 0;
        for (int i = 0; i < kNsMats; ++i) {
            first.at[i] = 0x7fffffff;
            if (i >= n) continue;
            ns_fill(*group[i], a, a.mat[i]);
            const int bytes = small_lds(a.mat[i].mp, a.mat[i].np);
            if (bytes > lds) lds = bytes;
            first.at[i] = grid;
            grid += a.mat[i].batch;
        }
        if (!ns_lds((const void*)ns_small_kernel<T, MUON>, small_lds(64, 192), who)) return DGG_ERR_LAUNCH;
        hipLaunchKernelGGL((ns_small_kernel<T, MUON>), dim3(grid), dim3(kSmallThreads), lds, st, a, first);
    }
    for (int at = 0, n; (n = ns_group(mats, count, routes, kNarrowRoute, at, group)) > 0;) {
        NsFirst first;
        int lds;
        size_t bytes;
        const dim3 grid(ns_narrow_plan(group, n, a, first, lds, bytes)), block(kNarrowThreads);
        if (!ns_lds((const void*)ns_narrow_first_kernel<T, MUON>, narrow_lds(64), who) ||
            !ns_lds((const void*)ns_narrow_kernel<T, MUON>, narrow_lds(64), who))
            return DGG_ERR_LAUNCH;
        hipLaunchKernelGGL((ns_narrow_first_kernel<T, MUON>), grid, block, lds, st, a, first);
        for (int k = 0; k < steps; ++k) hipLaunchKernelGGL((ns_narrow_kernel<T, MUON>), grid, block, lds, st, (const NsArgs*)ws, first, k);
    }
    for (int at = 0, n; (n = ns_group(mats, count, routes, kGeneral, at, group)) > 0;) {
        ns_plan(group, n, a, P);
        const dim3 block(kThreads);
        const NsArgs* args = (const NsArgs*)ws;
        hipLaunchKernelGGL((ns_norm_kernel<T, MUON>), dim3(P.grid[kNorm]), block, 0, st, a, P.first[kNorm]);
        hipLaunchKernelGGL((ns_split_kernel<T, MUON>), dim3(P.grid[kSplit]), block, 0, st, args, P.first[kSplit]);
        constexpr int lds1 = Prod<1, 3>::kLds, lds2 = Prod<2, 2>::kLds;
        for (int k = 0; k < steps; ++k) {
            hipLaunchKernelGGL((ns_gram_kernel<3>), dim3(P.grid[kGram]), block, lds1, st, args, P.first[kGram], k);
            if (P.grid[kSum]) hipLaunchKernelGGL(ns_sum_kernel, dim3(P.grid[kSum]), block, 0, st, args, P.first[kSum], k);
            hipLaunchKernelGGL((ns_square_kernel<3>), dim3(P.grid[kSquare]), block, lds1, st, args, P.first[kSquare], k);
            using Last = typename std::conditional<MUON, ToMuon, T>::type;
            const bool last = k + 1 == steps;
            const dim3 grid(P.grid[kApply]);
            const NsFirst& f = P.first[kApply];
            if (P.f_apply == 2) {
                if (last) hipLaunchKernelGGL((ns_apply_kernel<2, 2, Last>), grid, block, lds2, st, args, f, k);
                else hipLaunchKernelGGL((ns_apply_kernel<2, 2, void>), grid, block, lds2, st, args, f, k);
            } else {
                if (last) hipLaunchKernelGGL((ns_apply_kernel<1, 3, Last>), grid, block, lds1, st, args, f, k);
                else hipLaunchKernelGGL((ns_apply_kernel<1, 3, void>), grid, block, lds1, st, args, f, k);
            }
        }
    }
    return check_launch(who);
}

int64_t ns_ws(const dgg_matrix* mats, int count, const char* who) {
    const int rc = ns_check(mats, count, who);
    return rc != DGG_OK ? rc : ns_need(mats, count, who);
}

}  // namespace
}  // namespace dgg

using namespace dgg;

extern "C" {

int64_t dgg_orthogonalize_workspace_bytes(const dgg_matrix* mats, int count) {
    return ns_ws(mats, count, "dgg_orthogonalize_workspace_bytes");
}

int dgg_orthogonalize(const dgg_matrix* mats, int count, int dtype, const double* coefficients, int steps, double eps, void* ws,
                      size_t ws_bytes, void* stream) {
    const char* who = "dgg_orthogonalize";
    const int rc = ns_check(mats, count, who);
    if (rc != DGG_OK) return rc;
    if (dtype < DGG_F32 || dtype > DGG_F16) {
        set_error_text("%s: unknown type %d", who, dtype);
        return DGG_ERR_INVALID;
    }
    NsArgs a = {};
    a.eps = eps;
    hipStream_t st = (hipStream_t)stream;
    return dtype == DGG_F32 ? ns_run<float, false>(mats, count, a, coefficients, steps, ws, ws_bytes, st, who)
         : dtype == DGG_BF16 ? ns_run<__bf16, false>(mats, count, a, coefficients, steps, ws, ws_bytes, st, who)
                             : ns_run<_Float16, false>(mats, count, a, coefficients, steps, ws, ws_bytes, st, who);
}

int dgg_muon_step(const dgg_matrix* mats, int count, double lr, double momentum, int nesterov, double weight_decay, int adjust,
                  double grad_scale, const double* coefficients, int steps, double eps, void* ws, size_t ws_bytes, void* stream) {
    const char* who = "dgg_muon_step";
    const int rc = ns_check(mats, count, who);
    if (rc != DGG_OK) return rc;
    if (adjust < DGG_MUON_SPECTRAL || adjust > DGG_MUON_MATCH_RMS || !isfinite(lr) || !isfinite(momentum) || !isfinite(weight_decay) ||
        !isfinite(grad_scale)) {
        set_error_text("%s: unknown adjustment %d, or a hyper-parameter that is not finite", who, adjust);
        return DGG_ERR_INVALID;
    }
    NsArgs a = {};
    a.update = {(float)momentum, (float)grad_scale, nesterov != 0};
    a.lr = lr;
    a.adjust = adjust;
    a.decay = (float)(lr * weight_decay);
    a.eps = eps;
    return ns_run<float, true>(mats, count, a, coefficients, steps, ws, ws_bytes, (hipStream_t)stream, who);
}

}  // extern "C"
