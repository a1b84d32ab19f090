// Orthogonalisation of matrices by Newton-Schulz products, and the Muon step built on it.
//   X_0 = U / (|U|_F + eps);   X <- a X + B X,  B = b A + c A^2,  A = X X^T      over the shorter side, `steps` times
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
// two (exact: the factor that is left of 1 / (|U| + eps) goes into the first step's coefficients), and every later operand has
// a bound that follows from |X_0| and the coefficients (ns_bounds) and is scaled by a power of two to stay below 2^15.
//
// Layout.  All products are C[i][j] = sum_k P[i][k] Q[j][k] with k contiguous in both operands: A = X X^T from X stored by rows,
// A^2 from A (symmetric), B X from B and X stored by columns.  So X is kept in both layouts.  A row is cut into blocks of 32 k, a
// block is 128 bytes: 32 hi, 32 lo.  Both sizes are padded to multiples of 64 with zeros, which stay zeros in every product.
#include <math.h>

#include "dgg_internal.h"

namespace dgg {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) float lds_f32;
typedef __attribute__((address_space(3))) half8 lds_half8;

constexpr int kNsMats = 16;      // matrices (stacks of them) per launch
constexpr int kNsSteps = 16;
constexpr int kNsParts = 256;    // partial sums of squares per matrix, at most
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
    int at_norm, at_split, at_gram, at_sum, at_square, at_apply;   // first workgroup in each launch
};

// One step's coefficients and the bounds that follow from them (ns_bounds): |X| <= r, |b A + c A^2| <= mb, |X'| <= grow |X|
struct NsStep { float a, b, c, r, mb, grow; };

// The powers of two of one matrix in one step: X = planes * sx, planes of A, B and the next X = value * sa, sb, sx_next
struct NsScale { float sx, sa, sb, sx_next; };

struct NsArgs {
    NsMat mat[kNsMats];
    int count;
    char* ws;
    int dtype;               // of in / out
    int muon, nesterov;
    float mu, gscale, decay;
    int adjust;
    double lr, eps;
    int steps;
    NsStep step[kNsSteps];
    int k;                   // the current step
};

static_assert(sizeof(NsArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ const NsMat& find(const NsArgs& a, int NsMat::*at, int& local) {
    int d = 0;
    for (int i = 1; i < a.count; ++i)
        if ((int)blockIdx.x >= a.mat[i].*at) d = i;
    local = (int)blockIdx.x - a.mat[d].*at;
    return a.mat[d];
}

// bytes of one matrix' planes with r rows of k columns
__host__ __device__ __forceinline__ size_t plane_bytes(int r, int k) { return (size_t)r * k * 4; }
// halfs from the start of a row's planes to (hi of) column k; lo lies 32 further on
__device__ __forceinline__ int plane_at(int k) { return (k >> 5) * 64 + (k & 31); }

__device__ __forceinline__ float load_as_float(const void* p, long long i, int dtype) {
    if (dtype == DGG_F32) return ((const float*)p)[i];
    if (dtype == DGG_BF16) return (float)((const __bf16*)p)[i];
    return (float)((const _Float16*)p)[i];
}

__device__ __forceinline__ double block_sum(double v, double* sh /* kThreads / 64 */) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) s += sh[i];
    return s;
}

// u of the muon step from the gradient and the momentum AFTER its update
__device__ __forceinline__ float muon_u(const NsArgs& a, float g, float m) { return a.nesterov ? fmaf(a.mu, m, a.gscale * g) : m; }

// ------------------------------------------------------------------------------------------------ norm
// sum of squares in 64 bits, one partial a workgroup (muon: M is updated on the way)
__global__ __launch_bounds__(kThreads) void ns_norm_kernel(NsArgs a) {
    __shared__ double sh[kThreads / 64];
    int local;
    const NsMat& M = find(a, &NsMat::at_norm, local);
    const int bat = local / M.parts, part = local - bat * M.parts;
    const char* in = (const char*)M.in + (size_t)bat * M.in_stride * (a.dtype == DGG_F32 ? 4 : 2);
    float* mom = a.muon ? M.mom + (size_t)bat * M.mom_stride : nullptr;
    const long long total = (long long)M.rows * M.cols;
    double s = 0.0;
    for (long long e = (long long)part * kThreads + threadIdx.x; e < total; e += (long long)M.parts * kThreads) {
        const long long r = e / M.cols, c = e - r * M.cols;
        float u = load_as_float(in, r * M.ld_in + c, a.dtype);
        if (a.muon) {
            float* mp = mom + r * M.ld_mom + c;
            const float m = fmaf(a.mu, *mp, a.gscale * u);
            *mp = m;
            u = muon_u(a, u, m);
        }
        s = fma((double)u, (double)u, s);
    }
    s = block_sum(s, sh);
    if (threadIdx.x == 0) ((double*)(a.ws + M.part))[(size_t)bat * M.parts + part] = s;
}

// ------------------------------------------------------------------------------------------------ planes of X_0
__device__ __forceinline__ void split2(float x, _Float16& hi, _Float16& lo) {
    hi = (_Float16)x;
    lo = (_Float16)(x - (float)hi);
}

// the power of two that brings `bound` into [2^14, 2^15)
__device__ __forceinline__ float below(float bound) { return ldexpf(1.f, 14 - ilogbf(bound)); }

// 64 x 64 of X: U read along its rows, written by rows and by columns of X as planes of U * 2^k
__global__ __launch_bounds__(kThreads) void ns_split_kernel(NsArgs a) {
    __shared__ double sh[kThreads / 64];
    __shared__ float t[64][65];   // [i][j] of X
    int local;
    const NsMat& M = find(a, &NsMat::at_split, local);
    const int ti = M.mp / 64, tj = M.np / 64;
    const int bat = local / (ti * tj), tile = local - bat * ti * tj, i0 = tile / tj * 64, j0 = tile % tj * 64;
    double s = 0.0;
    for (int p = threadIdx.x; p < M.parts; p += kThreads) s += ((const double*)(a.ws + M.part))[(size_t)bat * M.parts + p];
    const double norm = sqrt(block_sum(s, sh));
    // 2^k |U| in [2^14, 2^15): no element of the planes is larger.  A zero, infinite or NaN norm keeps k = 0.
    const int k = norm > 0.0 && norm < INFINITY ? 14 - ilogb(norm) : 0;
    if (tile == 0 && threadIdx.x == 0) {
        // every operand's bound: the one of the coefficients, or, for a norm far below eps, what |X_0| can have grown to
        NsScale* o = (NsScale*)(a.ws + M.scal) + (size_t)bat * kNsSteps;
        float r = (float)(norm / (norm + a.eps));
        if (!(r > 0x1p-40f)) r = 0x1p-40f;
        float sx = (float)(1.0 / ldexp(norm + a.eps, k));
        for (int i = 0; i < a.steps; ++i) {
            const NsStep& S = a.step[i];
            r = fminf(1.01f * r, S.r);
            const float next = S.grow * r;
            NsScale z;
            z.sx = sx;
            z.sa = below(r * r);
            z.sb = below(fmaxf(fminf(S.mb, (fabsf(S.b) + fabsf(S.c) * r * r) * r * r), 0x1p-100f));
            z.sx_next = below(i + 1 < a.steps ? fminf(next, a.step[i + 1].r) : next);
            o[i] = z;
            sx = 1.f / z.sx_next;
            r = next;
        }
    }
    const char* in = (const char*)M.in + (size_t)bat * M.in_stride * (a.dtype == DGG_F32 ? 4 : 2);
    const float* mom = a.muon ? M.mom + (size_t)bat * M.mom_stride : nullptr;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r0 = M.turned ? j0 : i0, c0 = M.turned ? i0 : j0;   // of U
    for (int q = wave; q < 64; q += 4) {
        const int r = r0 + q, c = c0 + lane;
        float u = 0.f;
        if (r < M.rows && c < M.cols) {
            u = load_as_float(in, (long long)r * M.ld_in + c, a.dtype);
            if (a.muon) u = muon_u(a, u, mom[(long long)r * M.ld_mom + c]);
            u = (float)ldexp((double)u, k);
        }
        if (M.turned) t[lane][q] = u;
        else t[q][lane] = u;
    }
    __syncthreads();
    _Float16* xr = (_Float16*)(a.ws + M.xr + (size_t)bat * plane_bytes(M.mp, M.np));
    _Float16* xt = (_Float16*)(a.ws + M.xt + (size_t)bat * 2 * plane_bytes(M.np, M.mp));
    // 64 rows of 64 k: 8 k a thread, twice per layout
    for (int q = threadIdx.x; q < 512; q += kThreads) {
        const int row = q >> 3, k8 = (q & 7) * 8;
        half8 hi, lo, thi, tlo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 h, l;
            split2(t[row][k8 + e], h, l);
            hi[e] = h; lo[e] = l;
            split2(t[k8 + e][row], h, l);
            thi[e] = h; tlo[e] = l;
        }
        _Float16* o = xr + (size_t)(i0 + row) * M.np * 2 + plane_at(j0 + k8);
        *(half8*)o = hi;
        *(half8*)(o + 32) = lo;
        o = xt + (size_t)(j0 + row) * M.mp * 2 + plane_at(i0 + k8);
        *(half8*)o = thi;
        *(half8*)(o + 32) = tlo;
    }
}

// ------------------------------------------------------------------------------------------------ product
// acc[64 x 64 per wave: 2 x 2 blocks of 32 x 32] of C[i][j] = sum_k P[i][k] Q[j][k], TM x TN = 32 fi * 2 x 32 fj * 2 per workgroup,
// waves 2 x 2.  P, Q: row 0's planes; rows beyond the last are read as the last (their results are not stored).
// LDS: two stages of (TM + TN) rows x 128 bytes.  The 16-byte chunk q of row r lies at chunk q ^ ((r >> 1) & 7): a fragment's 16
// rows then fall on 16 different groups of banks.  The swizzle is in the GLOBAL address: LDS-DMA writes lane by lane.
template <int FI, int FJ>
struct Prod {
    static constexpr int TM = 64 * FI, TN = 64 * FJ, kStage = (TM + TN) * 128;
    static constexpr int kLds = 2 * kStage;

    __device__ static __forceinline__ void run(const char* P, int prow, int prows, const char* Q, int qrow, int qrows,
                                               size_t pitch, int kb0, int kb1, f32x16 (&acc)[FI][FJ]) {
        extern __shared__ char smem[];
        const unsigned lds = (unsigned)(size_t)(lds_char*)smem;
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wi = wave >> 1, wj = wave & 1;
        const int c = tid & 7, rr = tid >> 3;
        constexpr int NP = TM / 32, NQ = TN / 32;
        const char* src[NP + NQ];
#pragma unroll
        for (int t = 0; t < NP + NQ; ++t) {
            const int row = (t < NP ? t : t - NP) * 32 + rr;
            const int at = t < NP ? min(prow + row, prows - 1) : min(qrow + row, qrows - 1);
            src[t] = (t < NP ? P : Q) + (size_t)at * pitch + (size_t)((c ^ ((row >> 1) & 7)) * 16);
        }
        auto fetch = [&](int kb, int stage) {
#pragma unroll
            for (int t = 0; t < NP + NQ; ++t)
                __builtin_amdgcn_global_load_lds(
                    reinterpret_cast<const float*>(src[t] + (size_t)kb * 128),
                    (lds_f32*)(size_t)__builtin_amdgcn_readfirstlane(lds + stage * kStage + t * 4096 + wave * 1024), 16, 0, 0);
        };
        const int fr = lane & 31, fk = lane >> 5;
        auto frag = [&](int stage, int base_row, int plane, int kk) {
            const int row = base_row + fr, chunk = (plane * 4 + kk * 2 + fk) ^ ((row >> 1) & 7);
            return *(lds_half8*)(size_t)(lds + stage * kStage + row * 128 + chunk * 16);
        };
        fetch(kb0, 0);
        for (int kb = kb0; kb < kb1; ++kb) {
            const int st = (kb - kb0) & 1;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this stage's pieces have landed (LDS-DMA is counted by vmcnt)
            __syncthreads();                                   // .. everyone's; and everyone is done with the other stage
            if (kb + 1 < kb1) fetch(kb + 1, st ^ 1);
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                half8 ph[FI], pl[FI], qh[FJ], ql[FJ];
#pragma unroll
                for (int i = 0; i < FI; ++i) {
                    ph[i] = frag(st, (wi * FI + i) * 32, 0, kk);
                    pl[i] = frag(st, (wi * FI + i) * 32, 1, kk);
                }
#pragma unroll
                for (int j = 0; j < FJ; ++j) {
                    qh[j] = frag(st, TM + (wj * FJ + j) * 32, 0, kk);
                    ql[j] = frag(st, TM + (wj * FJ + j) * 32, 1, kk);
                }
#pragma unroll
                for (int i = 0; i < FI; ++i)
#pragma unroll
                    for (int j = 0; j < FJ; ++j) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], ql[j], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl[i], qh[j], acc[i][j], 0, 0, 0);
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph[i], qh[j], acc[i][j], 0, 0, 0);
                    }
            }
        }
    }

    // calls f(i, j, v) for the thread's elements, four consecutive i at a time: v[0..3] at rows i .. i + 3, column j
    template <typename F> __device__ static __forceinline__ void each(const f32x16 (&acc)[FI][FJ], F f) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int j = 0; j < FJ; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
                    f((wi * FI + i) * 32 + 8 * q + 4 * (lane >> 5), (wj * FJ + j) * 32 + (lane & 31), v);
                }
    }
};

template <int FI, int FJ> __device__ __forceinline__ void zero(f32x16 (&acc)[FI][FJ]) {
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
}

// tile number -> (ti, tj) with ti <= tj, of a t x t grid, row by row
__device__ __forceinline__ void upper(int tile, int t, int& ti, int& tj) {
    ti = 0;
    while (tile >= t - ti) {
        tile -= t - ti;
        ++ti;
    }
    tj = ti + tile;
}

__device__ __forceinline__ NsScale scale_of(const NsArgs& a, const NsMat& M, int bat) {
    return ((const NsScale*)(a.ws + M.scal))[(size_t)bat * kNsSteps + a.k];
}

// four values at rows i .. i + 3 of column j into planes stored by columns (row j, k = i ..): 8 bytes each
__device__ __forceinline__ void store_planes_t(_Float16* base, size_t pitch, int i, int j, const float (&v)[4]) {
    half4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        _Float16 h, l;
        split2(v[e], h, l);
        hi[e] = h;
        lo[e] = l;
    }
    _Float16* o = base + (size_t)j * pitch + plane_at(i);
    *(half4*)o = hi;
    *(half4*)(o + 32) = lo;
}
// .. and stored by rows (row i + e, k = j)
__device__ __forceinline__ void store_planes(_Float16* base, size_t pitch, int i, int j, const float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        _Float16 h, l;
        split2(v[e], h, l);
        _Float16* o = base + (size_t)(i + e) * pitch + plane_at(j);
        o[0] = h;
        o[32] = l;
    }
}
__device__ __forceinline__ float load_plane(const _Float16* base, size_t pitch, int r, int k) {
    const _Float16* p = base + (size_t)r * pitch + plane_at(k);
    return (float)p[0] + (float)p[32];
}

// A = X X^T, tiles on and above the diagonal, a range of k each: fp32 slabs [split][mp][mp]
template <int F>
__global__ __launch_bounds__(kThreads) void ns_gram_kernel(NsArgs a) {
    int local;
    const NsMat& M = find(a, &NsMat::at_gram, local);
    const int t = (M.mp + 64 * F - 1) / (64 * F), tiles = t * (t + 1) / 2, per = tiles * M.splits;
    const int bat = local / per, rest = local - bat * per, split = rest / tiles;
    int ti, tj;
    upper(rest - split * tiles, t, ti, tj);
    const char* x = a.ws + M.xr + (size_t)bat * plane_bytes(M.mp, M.np);
    f32x16 acc[F][F];
    zero(acc);
    const int kb0 = split * M.kblocks, kb1 = min(kb0 + M.kblocks, M.np / 32);
    Prod<F, F>::run(x, ti * 64 * F, M.mp, x, tj * 64 * F, M.mp, (size_t)M.np * 4, kb0, kb1, acc);
    float* slab = (float*)(a.ws + M.slab) + ((size_t)bat * M.splits + split) * M.mp * M.mp;
    Prod<F, F>::each(acc, [&](int i, int j, const float (&v)[4]) {
        i += ti * 64 * F;
        j += tj * 64 * F;
        if (j >= M.mp) return;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < M.mp) slab[(size_t)(i + e) * M.mp + j] = v[e];
    });
}

// sums the slabs in order: planes of A, both triangles; 32 x 32 elements a workgroup
__global__ __launch_bounds__(kThreads) void ns_sum_kernel(NsArgs a) {
    __shared__ float t[32][33];
    int local;
    const NsMat& M = find(a, &NsMat::at_sum, local);
    const int n32 = M.mp / 32, tiles = n32 * (n32 + 1) / 2, bat = local / tiles;
    int ti, tj;
    upper(local - bat * tiles, n32, ti, tj);
    const NsScale z = scale_of(a, M, bat);
    const float* slab = (const float*)(a.ws + M.slab) + (size_t)bat * M.splits * M.mp * M.mp;
    _Float16* A = (_Float16*)(a.ws + M.a + (size_t)bat * plane_bytes(M.mp, M.mp));
    const int c = threadIdx.x & 31;
    for (int r = threadIdx.x >> 5; r < 32; r += 8) {
        const size_t at = (size_t)(ti * 32 + r) * M.mp + tj * 32 + c;
        float v = 0.f;
        for (int sp = 0; sp < M.splits; ++sp) v += slab[(size_t)sp * M.mp * M.mp + at];
        t[r][c] = v * z.sx * z.sx * z.sa;   // (in this order: sx * sx alone may be below fp32's range)
    }
    __syncthreads();
    // a 32 x 32 block is one 128-byte piece of each row: 4 threads x 8 k of hi and lo; then the block's mirror image
    const int row = threadIdx.x >> 2, k8 = (threadIdx.x & 3) * 8;
    if (row < 64) {
        const int r = row & 31, mirror = row >> 5;
        half8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 h, l;
            split2(mirror || (ti == tj && k8 + e < r) ? t[k8 + e][r] : t[r][k8 + e], h, l);
            hi[e] = h;
            lo[e] = l;
        }
        if (!mirror || ti != tj) {
            _Float16* o = A + (size_t)((mirror ? tj : ti) * 32 + r) * M.mp * 2 + (mirror ? ti : tj) * 64 + k8;
            *(half8*)o = hi;
            *(half8*)(o + 32) = lo;
        }
    }
}

// B = b A + c A^2, tiles on and above the diagonal and their mirror images
template <int F>
__global__ __launch_bounds__(kThreads) void ns_square_kernel(NsArgs a) {
    int local;
    const NsMat& M = find(a, &NsMat::at_square, local);
    const int t = (M.mp + 64 * F - 1) / (64 * F), tiles = t * (t + 1) / 2, bat = local / tiles;
    int ti, tj;
    upper(local - bat * tiles, t, ti, tj);
    const _Float16* A = (const _Float16*)(a.ws + M.a + (size_t)bat * plane_bytes(M.mp, M.mp));
    _Float16* B = (_Float16*)(a.ws + M.b + (size_t)bat * plane_bytes(M.mp, M.mp));
    f32x16 acc[F][F];
    zero(acc);
    Prod<F, F>::run((const char*)A, ti * 64 * F, M.mp, (const char*)A, tj * 64 * F, M.mp, (size_t)M.mp * 4, 0, M.mp / 32, acc);
    const NsScale z = scale_of(a, M, bat);
    const float ratio = z.sb / z.sa, fb = a.step[a.k].b * ratio, fc = a.step[a.k].c * ratio / z.sa;
    const size_t pitch = (size_t)M.mp * 2;
    Prod<F, F>::each(acc, [&](int i, int j, const float (&v)[4]) {
        i += ti * 64 * F;
        j += tj * 64 * F;
        if (i >= M.mp || j >= M.mp) return;
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = fmaf(fc, v[e], fb * load_plane(A, pitch, j, i + e));
        if (ti != tj) store_planes_t(B, pitch, i, j, w);
        store_planes(B, pitch, i, j, w);
    });
}

__device__ __forceinline__ void store_as(void* p, long long i, float v, int dtype) {
    if (dtype == DGG_F32) ((float*)p)[i] = v;
    else if (dtype == DGG_BF16) ((__bf16*)p)[i] = (__bf16)v;
    else ((_Float16*)p)[i] = (_Float16)v;
}

// X <- a X + B X: planes in both layouts, or (last step) the result
template <int FI, int FJ>
__global__ __launch_bounds__(kThreads) void ns_apply_kernel(NsArgs a) {
    int local;
    const NsMat& M = find(a, &NsMat::at_apply, local);
    using Pr = Prod<FI, FJ>;
    const int ti = (M.mp + Pr::TM - 1) / Pr::TM, tj = (M.np + Pr::TN - 1) / Pr::TN;
    const int bat = local / (ti * tj), tile = local - bat * ti * tj, i0 = tile % ti * Pr::TM, j0 = tile / ti * Pr::TN;
    const char* B = a.ws + M.b + (size_t)bat * plane_bytes(M.mp, M.mp);
    const size_t xtb = plane_bytes(M.np, M.mp);
    const int flip = a.k & 1;   // which half of xt holds X
    const _Float16* xt = (const _Float16*)(a.ws + M.xt + ((size_t)bat * 2 + flip) * xtb);
    _Float16* xt_next = (_Float16*)(a.ws + M.xt + ((size_t)bat * 2 + (flip ^ 1)) * xtb);
    _Float16* xr = (_Float16*)(a.ws + M.xr + (size_t)bat * plane_bytes(M.mp, M.np));
    f32x16 acc[FI][FJ];
    zero(acc);
    Pr::run(B, i0, M.mp, (const char*)xt, j0, M.np, (size_t)M.mp * 4, 0, M.mp / 32, acc);
    const NsScale z = scale_of(a, M, bat);
    const float fx = a.step[a.k].a * z.sx, fb = z.sx / z.sb;
    const size_t pt = (size_t)M.mp * 2, pr = (size_t)M.np * 2;
    const size_t es = a.dtype == DGG_F32 ? 4 : 2;
    char* out = (char*)M.out + (size_t)bat * M.out_stride * es;
    Pr::each(acc, [&](int i, int j, const float (&v)[4]) {
        i += i0;
        j += j0;
        if (i >= M.mp || j >= M.np) return;
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf(fb, v[e], fx * load_plane(xt, pt, j, i + e));
        if (a.k + 1 < a.steps) {
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] *= z.sx_next;
            store_planes_t(xt_next, pt, i, j, y);
            store_planes(xr, pr, i, j, y);
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i + e >= M.m || j >= M.n) continue;
            const long long at = M.turned ? (long long)j * M.ld_out + i + e : (long long)(i + e) * M.ld_out + j;
            if (a.muon) {
                float* w = (float*)out + at;
                *w = fmaf(-M.step, y[e], a.decay * *w);
            } else {
                store_as(out, at, y[e], a.dtype);
            }
        }
    });
}

// ------------------------------------------------------------------------------------------------ host side
// Bounds of every step's operands from the coefficients alone.  |X_0| <= 1 in the 2-norm; with r = |X| the singular values lie in
// [0, r], so |A| <= r^2, |B| <= max |b s^2 + c s^4|, |X'| <= max |a s + b s^3 + c s^5| over [0, r], and no element exceeds its
// matrix' norm.  1 % is added for the roundings.
bool ns_bounds(const double* coef, int steps, NsStep* out) {
    double r = 1.0;
    for (int k = 0; k < steps; ++k) {
        const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
        r *= 1.01;
        double mb = 0.0, mx = 0.0, mg = 0.0;
        for (int i = 0; i <= 4096; ++i) {
            const double s = r * i / 4096.0, s2 = s * s, g = a + b * s2 + c * s2 * s2;
            mb = fmax(mb, fabs(b * s2 + c * s2 * s2));
            mx = fmax(mx, fabs(s * g));
            mg = fmax(mg, fabs(g));
        }
        mb *= 1.01;
        mx *= 1.01;
        if (!isfinite(a + b + c) || !(mb < 1e6) || !(mx < 1e6) || !(mx > 1e-6) || !(mg < 1e6)) return false;
        out[k] = {(float)a, (float)b, (float)c, (float)r, (float)fmax(mb, 1e-6), (float)(1.01 * mg)};
        r = mx;
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

// Sizes, workspace places and first workgroups of up to kNsMats matrices; returns the workspace bytes.
size_t ns_plan(const dgg_matrix* mats, int count, NsArgs& a, int grids[6]) {
    size_t at = 0;
    for (int k = 0; k < 6; ++k) grids[k] = 0;
    a.count = count;
    for (int i = 0; i < count; ++i) {
        const dgg_matrix& in = mats[i];
        NsMat& M = a.mat[i];
        M.in = in.in; M.out = in.out; M.mom = in.momentum;
        M.in_stride = in.in_stride; M.out_stride = in.out_stride; M.mom_stride = in.momentum_stride;
        M.ld_in = in.ld_in; M.ld_out = in.ld_out; M.ld_mom = in.ld_momentum;
        M.rows = in.rows; M.cols = in.cols; M.batch = (int)in.batch;
        M.turned = in.rows > in.cols;
        M.m = M.turned ? in.cols : in.rows;
        M.n = M.turned ? in.rows : in.cols;
        M.mp = ceil_div(M.m, 64) * 64;
        M.np = ceil_div(M.n, 64) * 64;
        const double f = a.adjust == DGG_MUON_SPECTRAL ? sqrt(fmax(1.0, (double)in.rows / in.cols)) : 0.2 * sqrt((double)M.n);
        M.step = (float)(a.lr * f);
        M.parts = ceil_div((long long)M.m * M.n, kThreads * 16);
        if (M.parts > kNsParts) M.parts = kNsParts;
        const int t = ceil_div(M.mp, 128), tiles = t * (t + 1) / 2;
        int splits = ceil_div(128, (long long)tiles * M.batch);
        if (splits > M.np / 256) splits = M.np / 256;
        if (splits < 1) splits = 1;
        M.kblocks = ceil_div(M.np / 32, splits);
        M.splits = ceil_div(M.np / 32, M.kblocks);
        const size_t b = (size_t)M.batch;
        M.xr = at;   at = up(at + b * plane_bytes(M.mp, M.np));
        M.xt = at;   at = up(at + b * 2 * plane_bytes(M.np, M.mp));
        M.a = at;    at = up(at + b * plane_bytes(M.mp, M.mp));
        M.b = at;    at = up(at + b * plane_bytes(M.mp, M.mp));
        M.slab = at; at = up(at + b * M.splits * M.mp * M.mp * 4);
        M.part = at; at = up(at + b * M.parts * 8);
        M.scal = at; at = up(at + b * kNsSteps * sizeof(NsScale));
        const int n32 = M.mp / 32;
        int* first[6] = {&M.at_norm, &M.at_split, &M.at_gram, &M.at_sum, &M.at_square, &M.at_apply};
        const int blocks[6] = {M.parts, (M.mp / 64) * (M.np / 64), tiles * M.splits, n32 * (n32 + 1) / 2, tiles,
                               t * ceil_div(M.np, 128)};
        for (int k = 0; k < 6; ++k) {
            *first[k] = grids[k];
            grids[k] += blocks[k] * M.batch;
        }
    }
    return at;
}

int ns_run(const dgg_matrix* mats, int count, NsArgs& a, const double* coef, int steps, void* ws, size_t ws_bytes,
           hipStream_t st, const char* who) {
    if (steps < 1 || steps > kNsSteps || !coef || !(a.eps >= 0.0) || !ns_bounds(coef, steps, a.step)) {
        set_error_text("%s: 1 .. %d steps, eps >= 0 and coefficients whose iterates stay bounded (|X| < 1e6) are needed", who, kNsSteps);
        return DGG_ERR_INVALID;
    }
    for (int i = 0; i < count; ++i) {
        const dgg_matrix& m = mats[i];
        const bool mom = !a.muon || (m.momentum && m.ld_momentum >= m.cols && m.momentum_stride >= 0);
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
    int g[6];
    for (int at = 0; at < count; at += kNsMats)
        if (ns_plan(mats + at, count - at < kNsMats ? count - at : kNsMats, a, g) > ws_bytes) {
            set_error_text("%s: the workspace of %zu bytes is too small", who, ws_bytes);
            return DGG_ERR_WORKSPACE;
        }
    for (int at = 0; at < count; at += kNsMats) {
        ns_plan(mats + at, count - at < kNsMats ? count - at : kNsMats, a, g);
        const dim3 block(kThreads);
        hipLaunchKernelGGL(ns_norm_kernel, dim3(g[0]), block, 0, st, a);
        hipLaunchKernelGGL(ns_split_kernel, dim3(g[1]), block, 0, st, a);
        for (int k = 0; k < steps; ++k) {
            a.k = k;
            hipLaunchKernelGGL((ns_gram_kernel<2>), dim3(g[2]), block, (Prod<2, 2>::kLds), st, a);
            hipLaunchKernelGGL(ns_sum_kernel, dim3(g[3]), block, 0, st, a);
            hipLaunchKernelGGL((ns_square_kernel<2>), dim3(g[4]), block, (Prod<2, 2>::kLds), st, a);
            hipLaunchKernelGGL((ns_apply_kernel<2, 2>), dim3(g[5]), block, (Prod<2, 2>::kLds), st, a);
        }
    }
    return check_launch(who);
}

int64_t ns_ws(const dgg_matrix* mats, int count, const char* who) {
    const int rc = ns_check(mats, count, who);
    if (rc != DGG_OK) return rc;
    size_t need = 0;
    for (int at = 0; at < count; at += kNsMats) {
        NsArgs a = {};
        int g[6];
        const size_t n = ns_plan(mats + at, count - at < kNsMats ? count - at : kNsMats, a, g);
        if (n > need) need = n;
    }
    return (int64_t)need;
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
    a.dtype = dtype;
    a.eps = eps;
    return ns_run(mats, count, a, coefficients, steps, ws, ws_bytes, (hipStream_t)stream, who);
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
    a.dtype = DGG_F32;
    a.muon = 1;
    a.nesterov = nesterov != 0;
    a.mu = (float)momentum;
    a.gscale = (float)grad_scale;
    a.lr = lr;
    a.adjust = adjust;
    a.decay = (float)(1.0 - lr * weight_decay);
    a.eps = eps;
    return ns_run(mats, count, a, coefficients, steps, ws, ws_bytes, (hipStream_t)stream, who);
}

}  // extern "C"
