// Group normalisation with an activation over channels-last data: x (N, S, C), S points (rows) of C channels per sample,
// G groups of D = C / G channels.
//   forward   mean, var over the S x D elements of (n, g);  xh = (x - mean) rstd;  z = w[c] xh + b[c];  y = act(z)
//   backward  dz = dy act'(z);  dw[c] = sum_{n,s} dz xh;  db[c] = sum_{n,s} dz;
//             dx = rstd (w dz - mean(w dz) - xh mean(w dz xh))          (means over the group)
// act: none, LeakyReLU(slope) — the ResBlock's — or SiLU.
//
// Bound: HBM (2 E elements forward, 3 E backward), a few dozen vector instructions per 16 bytes beside it.
//
// Arithmetic.  Statistics are accumulated in 64 bits, and so is the pre-activation z = (x - mean) rstd w + b: its
// SIGN decides which side of LeakyReLU's kink an element lies on, i.e. a factor 1 / slope in its gradient, and an fp32 z
// would take the wrong side for every element within its rounding error of zero.  (64-bit vector instructions run at the
// rate of the fp32 ones here; per element they are 4 to 6 of them.)  What follows the sign is fp32, rounded once to the output
// type; dx of a group of a few elements is 64-bit to the end (grad_few).  SiLU and no activation have no such sign: they share
// the arithmetic, which keeps x - mean exact for data far from zero, at the price of those instructions.
//
// Three routes, chosen by gn_plan (us of a call's launches in a graph, inputs that change from pass to pass):
//  * "unit": a group's S x D elements fit the registers of at most one wave, or, long rows, of a workgroup.  L = 2^k lanes own one
//    (n, g): one read of x, mean and centred variance by lane shuffles.  1024 x 512 f32 in 32 groups: 3.5 us forward, 8.8 backward with dw
//    and db (launches); 16384 x 512: 19 and 27 us (3.5 and 3.7 TB/s); 8192 x 4096 bf16 in one group 50 and 72.
//  * "resident": a sample's points in a block of groups fit a workgroup's registers: one read, one launch.  128 x 2048 x 256 bf16
//    in 32 groups: 69 us forward (3.9 TB/s), 128 backward (3.2 TB/s: the arithmetic and the memory take turns, one workgroup a CU).
//  * "tile": a workgroup owns a range of the rows of one sample and a block of channels (a thread keeps ITS channels while
//    it walks down the rows), leaves per-channel partial sums in the workspace, and a small launch merges them in a fixed
//    order into the groups' statistics (and dw, db); a last launch applies them.  No atomics: results do not depend on the
//    order in which workgroups run.  30 x 1000 x 1020 bf16 in 60 groups: 50 and 87 us (x is read twice, dy too).
#include <type_traits>

#include "dgg_internal.h"

namespace dgg {
namespace {

constexpr int kGnThreads = 256;
constexpr int kMergeThreads = 1024;
constexpr int kGnFew = 8;   // elements of a group, at most, whose dx may be what cancellation leaves (grad_few)

// V elements of memory, one access at any address that an element may have (global memory is accessed unaligned): rows of any pitch
template <typename T, int V> struct Vec { T e[V]; };
template <int N> struct Bits { typedef uint32_t Type __attribute__((ext_vector_type(N / 4))); };
template <> struct Bits<4> { typedef uint32_t Type; };
template <> struct Bits<2> { typedef uint16_t Type; };

template <typename T, int V> __device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
    const Vec<T, V> r = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)r.e[i];
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.e[i] = (T)v[i];   // the one rounding to the output type (nearest even)
    *reinterpret_cast<Vec<T, V>*>(p) = r;
}

// Vector v of a group of `width` >= V channels: its first channel, and how many of its elements belong to the vector before it.  EVEN: V
// divides the width; else the last vector ends with the group, and what it shares with the one before is the same in both.
template <int V, bool EVEN> struct Span {
    int at, skip;
    __device__ __forceinline__ Span(int v, int width) : at(EVEN ? v * V : min(v * V, width - V)), skip(EVEN ? 0 : v * V - at) {}
};
__host__ __device__ __forceinline__ int vectors(int width, int V) { return (width + V - 1) / V; }

// 1 / (1 + exp(-z)) by the hardware's exp2 and reciprocal (1 unit in the last place each).  The exponent is formed in 64 bits and
// rounded once, so from z = -87 on the result is off by (|z| + 6) 2^-24 of itself at most; below, where it leaves fp32's normal numbers, it
// may be 0 (off by 2e-38).  (With expf and a division, 30 instructions an element,
// a forward pass over 64 M bf16 elements was bound by them: 77 us for the launch that moves 268 MB.)
__device__ __forceinline__ float sigmoid(double z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f((float)(z * -1.4426950408889634)));
}
// act(z) and act'(z) of a 64-bit pre-activation
__device__ __forceinline__ float act_value(double z, int act, float slope) {
    const float zf = (float)z;
    if (act == DGG_ACT_LEAKY_RELU) return z > 0.0 ? zf : zf * slope;
    if (act == DGG_ACT_SILU) return zf * sigmoid(z);
    return zf;
}
__device__ __forceinline__ float act_slope(double z, int act, float slope) {
    if (act == DGG_ACT_LEAKY_RELU) return z > 0.0 ? 1.f : slope;
    if (act == DGG_ACT_SILU) {
        const float zf = (float)z, s = sigmoid(z);
        return s * (1.f + zf * (1.f - s));
    }
    return 1.f;
}

// dx in a group of up to kGnFew elements, d = x - mean, m1 = mean(w dz), k2 = -rstd mean(w dz xh): the three terms cancel — to 0 for one
// element, to eps / (var + eps) of them for two —, so they are added up in 64 bits and rounded once; one element gives exactly 0.
__device__ __forceinline__ float grad_few(double d, float dz, float w, double rstd, double m1, double k2) {
    return (float)(rstd * fma(d, k2, fma((double)w, (double)dz, -m1)));
}

// V consecutive channels of weight or bias, or what stands for one that is not there (one branch for all of them)
template <int V> __device__ __forceinline__ void load_param(const float* p, long long c, float none, float (&v)[V]) {
    if (p) {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = p[c + k];
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = none;
    }
}

struct GnArgs {
    const void* x;
    const void* dy;
    void* out;              // y (forward) or dx (backward), contiguous
    const float* w;         // NULL: 1
    const float* b;         // NULL: 0
    double* stats;          // [N][G][2]: mean, rstd
    double* part;           // tile: [N][chunks][C][2]; unit backward: float [rows of partials][C][2]
    double* chan;           // tile backward: [N][C][2], part summed over the chunks (part itself where there is one)
    double* coef;           // tile backward: [N][G][2]: mean(w dz), mean(w dz xh)
    double* ranges;         // [ranges][C][2]: gn_param_grad
    float* dw;
    float* db;
    long long x_sn, x_ss, dy_sn, dy_ss;   // strides in elements; the channel stride is 1
    long long N, S;
    int C, G, D;
    int act;
    float slope;
    double eps;
    int chunks;             // tile: row ranges per sample
    long long chunk_rows;
    int tx;                 // tile: vectors of a row a workgroup covers
    int lanes;              // unit: lanes per group
    int blocks_g, blocks_n; // unit backward: grid; resident: blocks_g blocks of
    int res_groups;         // res_groups groups a sample
};

__device__ __forceinline__ double lane_sum(double v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// sum of v over the workgroup, in a fixed order, for every thread
__device__ __forceinline__ double block_sum(double v, double* sh /* blockDim.x / 64 */) {
    v = lane_sum(v, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) s += sh[i];
    return s;
}

// a lane's value summed over the lanes of its group: `lanes` of a wave, or (WIDE) the workgroup
template <bool WIDE> __device__ __forceinline__ double group_sum(double v, int lanes, double* sh /* WIDE: blockDim.x / 64 */) {
    if constexpr (WIDE) return block_sum(v, sh);
    else return lane_sum(v, lanes);
}

// Adds up the entries of n threads `stride` apart, y = 0 .. n - 1 the thread's own number among them, halving n: the first has the sum, in a
// fixed order.  sh: [N][blockDim.x], entry k of thread t at k * blockDim.x + t; every thread of the workgroup calls it.
template <int N> __device__ __forceinline__ void fold(double* sh, int y, int n, int stride) {
    __syncthreads();
    while (n > 1) {
        const int h = (n + 1) / 2;
        if (y < n - h)
#pragma unroll
            for (int k = 0; k < N; ++k) sh[k * blockDim.x + threadIdx.x] += sh[k * blockDim.x + threadIdx.x + h * stride];
        n = h;
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ unit route
template <typename T, int V, bool EVEN, int I, bool WIDE>
__global__ __launch_bounds__(kGnThreads) void gn_unit_fwd_kernel(GnArgs a) {
    __shared__ double wide[WIDE ? kGnThreads / 64 : 1];
    const int L = WIDE ? kGnThreads : a.lanes, lane = threadIdx.x & (L - 1);
    const long long u = ((long long)blockIdx.x * kGnThreads + threadIdx.x) / L;
    if (u >= a.N * a.G) return;   // whole groups of L lanes leave together: the shuffles below stay inside a group
    const unsigned n = (unsigned)u / (unsigned)a.G, g = (unsigned)u - n * (unsigned)a.G;
    const int dv = vectors(a.D, V), nv = (int)a.S * dv;
    const T* x = (const T*)a.x + (long long)n * a.x_sn + (long long)g * a.D;
    float v[I][V], w[I][V], b[I][V];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < I; ++i) {   // (lanes beyond the end: the last vector once more, not used)
        const int e = min(lane + i * L, nv - 1), s = a.S == 1 ? 0 : e / dv, cv = Span<V, EVEN>(e - s * dv, a.D).at;
        load_vec<T, V>(x + (long long)s * a.x_ss + cv, v[i]);
        load_param<V>(a.w, (long long)g * a.D + cv, 1.f, w[i]);
        load_param<V>(a.b, (long long)g * a.D + cv, 0.f, b[i]);
    }
    const auto skip = [&](int i) {   // elements of this lane's vector i that are not its own
        const int e = lane + i * L, s = a.S == 1 ? 0 : e / dv;
        return e < nv ? Span<V, EVEN>(e - s * dv, a.D).skip : V;
    };
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k >= skip(i)) sum += (double)v[i][k];
    const double count = (double)a.S * a.D;
    const double mean = group_sum<WIDE>(sum, L, wide) / count;   // (a constant group's mean is exact: z = bias there, not beside it)
    double m2 = 0.0;
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const double d = (double)v[i][k] - mean;
            if (k >= skip(i)) m2 = fma(d, d, m2);
        }
    const double rstd = 1.0 / sqrt(group_sum<WIDE>(m2, L, wide) / count + a.eps);
    if (a.stats && lane == 0) {
        a.stats[2 * u] = mean;
        a.stats[2 * u + 1] = rstd;
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
        const int e = lane + i * L;
        if (e >= nv) continue;
        const int s = a.S == 1 ? 0 : e / dv, c = (int)g * a.D + Span<V, EVEN>(e - s * dv, a.D).at;
        float y[V];
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = act_value(fma((double)v[i][k] - mean, rstd * (double)w[i][k], (double)b[i][k]), a.act, a.slope);
        store_vec<T, V>((T*)a.out + ((long long)n * a.S + s) * a.C + c, y);
    }
}

// Backward: a lane keeps its channels while it walks over the samples n, so that dw and db need no exchange between lanes until the
// end; every workgroup row leaves one partial per channel (64-bit sums, stored as fp32: 2^-24 of a partial for half the bytes).
// POINTS: S > 1, a lane has a vector of a point.
template <typename T, int V, bool EVEN, int I, bool WIDE, bool POINTS>
__global__ __launch_bounds__(kGnThreads) void gn_unit_bwd_kernel(GnArgs a) {
    __shared__ double wide[WIDE ? kGnThreads / 64 : 1];
    const int L = WIDE ? kGnThreads : a.lanes, lane = threadIdx.x & (L - 1), slot = threadIdx.x / L, slots = kGnThreads / L;
    const int per = a.G < slots ? slots / a.G : 1;             // samples side by side in a workgroup
    const int g = a.G < slots ? slot % a.G : (int)(blockIdx.x % a.blocks_g) * slots + slot;
    const int side = a.G < slots ? slot / a.G : 0;
    const bool on = side < per && g < a.G;
    const int nb = (int)(blockIdx.x / a.blocks_g);
    const int per_row = vectors(a.D, V), nv = POINTS ? (int)a.S * per_row : per_row;
    const auto point = [&](int e) { return POINTS ? e / per_row : 0; };
    const auto span = [&](int e) { return Span<V, EVEN>(e - point(e) * per_row, a.D); };
    float w[I][V], b[I][V];
    double dw[I][V], db[I][V];
#pragma unroll
    for (int i = 0; i < I; ++i) {
        const long long c = (long long)min(g, a.G - 1) * a.D + span(min(lane + i * L, nv - 1)).at;
        load_param<V>(a.w, c, 1.f, w[i]);
        load_param<V>(a.b, c, 0.f, b[i]);
#pragma unroll
        for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0.0;
    }
    const double inv = 1.0 / (POINTS ? (double)a.S * a.D : (double)a.D);
    const bool few = !WIDE && (POINTS ? a.S * a.D : a.D) <= kGnFew;
    for (long long n = on ? (long long)nb * per + side : a.N; n < a.N; n += (long long)a.blocks_n * per) {
        const T* x = (const T*)a.x + n * a.x_sn + (long long)g * a.D;
        const T* dy = (const T*)a.dy + n * a.dy_sn + (long long)g * a.D;
        const double mean = a.stats[2 * (n * a.G + g)], rstd = a.stats[2 * (n * a.G + g) + 1];
        float xv[I][V], dv[I][V];
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int e = min(lane + i * L, nv - 1), at = span(e).at;
            load_vec<T, V>(x + (POINTS ? point(e) * a.x_ss : 0) + at, xv[i]);
            load_vec<T, V>(dy + (POINTS ? point(e) * a.dy_ss : 0) + at, dv[i]);
        }
        double s1 = 0.0, s2 = 0.0;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int skip = lane + i * L < nv ? span(lane + i * L).skip : V;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const double d = (double)xv[i][k] - mean, xh = d * rstd;
                dv[i][k] *= act_slope(fma(xh, (double)w[i][k], (double)b[i][k]), a.act, a.slope);
                const double dz = (double)dv[i][k], wd = dz * (double)w[i][k];
                if (k >= skip) {
                    dw[i][k] = fma(dz, xh, dw[i][k]);
                    db[i][k] += dz;
                    s1 += wd;
                    s2 = fma(wd, xh, s2);
                }
            }
        }
        // dx = rstd ((w dz - m1) + (x - mean) k2).  Groups of more than a few elements: rstd w and the rest are rounded to fp32 and joined by
        // one fma (8192 x 4096 bf16 backward 66 us, 75 all in 64 bits)
        const double m1 = group_sum<WIDE>(s1, L, wide) * inv, k2 = -rstd * (group_sum<WIDE>(s2, L, wide) * inv);
        const double c1 = -rstd * m1, c2 = rstd * k2;
        const float fr = (float)rstd;
#pragma unroll
        for (int i = 0; i < I; ++i) {
            const int e = lane + i * L;
            if (e >= nv) continue;
            float o[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const double d = (double)xv[i][k] - mean;
                o[k] = few ? grad_few(d, dv[i][k], w[i][k], rstd, m1, k2) : fmaf(fr * w[i][k], dv[i][k], (float)fma(d, c2, c1));
            }
            store_vec<T, V>((T*)a.out + (POINTS ? n * a.S + point(e) : n) * a.C + g * a.D + span(e).at, o);
        }
    }
    if (!a.part) return;
    // the samples side by side are added up here: 1024 x 2048 f32 in one group left 17 MB of partial sums for 25 MB of data
    __shared__ double sh[WIDE ? 1 : kGnThreads * V * 2];
    float* p = (float*)a.part + 2ll * a.C * nb;
    if constexpr (POINTS) {   // first over the points, then over the samples
#pragma unroll
        for (int k = 0; k < V; ++k) {
            sh[(k * 2) * kGnThreads + threadIdx.x] = dw[0][k];
            sh[(k * 2 + 1) * kGnThreads + threadIdx.x] = db[0][k];
        }
        const int s = point(lane), first = lane < per_row;
        fold<2 * V>(sh, on && s < a.S ? s : (int)a.S, (int)a.S, per_row);
        fold<2 * V>(sh, on && first ? side : per, per, a.G * L);
        if (!on || side || !first) return;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            p[2 * (g * a.D + lane * V + k)] = (float)sh[(k * 2) * kGnThreads + threadIdx.x];
            p[2 * (g * a.D + lane * V + k) + 1] = (float)sh[(k * 2 + 1) * kGnThreads + threadIdx.x];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < I; ++i) {
        if (!WIDE && per > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < V; ++k) {
                sh[(k * 2) * kGnThreads + threadIdx.x] = dw[i][k];
                sh[(k * 2 + 1) * kGnThreads + threadIdx.x] = db[i][k];
            }
            __syncthreads();
            if (side == 0)
                for (int y = 1; y < per; ++y)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        dw[i][k] += sh[(k * 2) * kGnThreads + threadIdx.x + y * a.G * L];
                        db[i][k] += sh[(k * 2 + 1) * kGnThreads + threadIdx.x + y * a.G * L];
                    }
        }
        const int e = lane + i * L;
        const Span<V, EVEN> at = span(e);
        if (on && side == 0 && e < nv)
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (k >= at.skip) {
                    p[2 * (g * a.D + at.at + k)] = (float)dw[i][k];
                    p[2 * (g * a.D + at.at + k) + 1] = (float)db[i][k];
                }
    }
}

// ------------------------------------------------------------------------------------------------ tile route
// thread -> (vector of the row, row): tx vectors side by side, 256 / tx rows at a time; threads left over idle
struct Tile { int vx, ty, rows; bool on; };
__device__ __forceinline__ Tile tile_of(const GnArgs& a, int vecs, int by) {
    Tile t;
    t.rows = kGnThreads / a.tx;
    t.ty = threadIdx.x / a.tx;
    t.vx = by * a.tx + (int)threadIdx.x - t.ty * a.tx;
    t.on = t.ty < t.rows && t.vx < vecs;
    return t;
}

// sums a per-thread (p, q)[V] over the workgroup's rows; row 0 of each column holds the result
template <int V> __device__ __forceinline__ void column_sum(double (&p)[V], double (&q)[V], const GnArgs& a, const Tile& t) {
    __shared__ double sh[2 * V * kGnThreads];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        sh[2 * k * kGnThreads + threadIdx.x] = p[k];
        sh[(2 * k + 1) * kGnThreads + threadIdx.x] = q[k];
    }
    fold<2 * V>(sh, t.ty < t.rows ? t.ty : t.rows, t.rows, a.tx);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        p[k] = sh[2 * k * kGnThreads + threadIdx.x];
        q[k] = sh[(2 * k + 1) * kGnThreads + threadIdx.x];
    }
}

// load(s, v) and use(s, v) for the rows s, s + step, .. below s1, U loads ahead
template <int U, int N, typename Load, typename Use>
__device__ __forceinline__ void walk(long long s, long long s1, int step, Load load, Use use) {
    for (; s + (U - 1) * step < s1; s += U * step) {
        float v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) load(s + u * step, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) use(s + u * step, v[u]);
    }
    for (; s < s1; s += step) {
        float v[N];
        load(s, v);
        use(s, v);
    }
}

// per channel: sums of (x - k) and (x - k)^2 over a range of rows, k = the sample's first row: a shift that keeps the
// variance of data far from zero, removed again by gn_stats_kernel
template <typename T, int V>
__global__ __launch_bounds__(kGnThreads) void gn_tile_sum_kernel(GnArgs a) {
    const unsigned n = blockIdx.x / (unsigned)a.chunks, ch = blockIdx.x - n * (unsigned)a.chunks;
    const Tile t = tile_of(a, a.C / V, blockIdx.y);
    double p[V], q[V];
#pragma unroll
    for (int k = 0; k < V; ++k) p[k] = q[k] = 0.0;
    if (t.on) {
        const T* x = (const T*)a.x + (long long)n * a.x_sn + t.vx * V;
        const long long s0 = (long long)ch * a.chunk_rows, s1 = s0 + a.chunk_rows < a.S ? s0 + a.chunk_rows : a.S;
        float piv[V];
        load_vec<T, V>(x, piv);
        walk<4, V>(s0 + t.ty, s1, t.rows, [&](long long s, float (&v)[V]) { load_vec<T, V>(x + s * a.x_ss, v); },
                   [&](long long, float (&v)[V]) {
#pragma unroll
                       for (int k = 0; k < V; ++k) {
                           const double d = (double)v[k] - (double)piv[k];
                           p[k] += d;
                           q[k] = fma(d, d, q[k]);
                       }
                   });
    }
    column_sum<V>(p, q, a, t);
    if (t.on && t.ty == 0)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            double* o = a.part + 2ll * ((long long)blockIdx.x * a.C + t.vx * V + k);
            o[0] = p[k];
            o[1] = q[k];
        }
}

// The sums part[..][C][2] of one (n, g) over the row ranges, channel by channel: `use(c, p, q)` runs for each channel once, in one
// thread (T walkers a channel, added up in order).
template <typename Use> __device__ __forceinline__ void over_chunks(const GnArgs& a, const double* part, double* col /* 2 blockDim.x */, Use use) {
    const int wide = min(a.D, (int)blockDim.x), T = (int)blockDim.x / wide, w = (int)threadIdx.x / wide, c0 = (int)threadIdx.x - w * wide;
    for (int base = 0; base < a.D; base += wide) {
        const int c = base + c0;
        const bool on = w < T && c < a.D;
        double p = 0.0, q = 0.0;
        if (on) {
            const double* o = part + 2ll * c;
#pragma unroll 4
            for (int ch = w; ch < a.chunks; ch += T) {
                p += o[2ll * ch * a.C];
                q += o[2ll * ch * a.C + 1];
            }
        }
        __syncthreads();
        col[threadIdx.x] = p;
        col[blockDim.x + threadIdx.x] = q;
        fold<2>(col, w < T ? w : T, T, wide);
        if (on && w == 0) use(c, col[threadIdx.x], col[blockDim.x + threadIdx.x]);
    }
}

// One workgroup per (n, g) merges the shifted sums of its channels and row ranges: with d = x - k_c,
//   mean = (sum_c k_c + sum d / S) / D,   sum (x - mean)^2 = sum d^2 + 2 (k_c - mean) sum d + S sum_c (k_c - mean)^2
// (a channel's sums over the ranges take the place of its first range's between the two)
template <typename T>
__global__ __launch_bounds__(kMergeThreads) void gn_stats_kernel(GnArgs a) {
    __shared__ double sh[kMergeThreads / 64], col[kMergeThreads * 2];
    const unsigned n = blockIdx.x / (unsigned)a.G, g = blockIdx.x - n * (unsigned)a.G;
    const T* x0 = (const T*)a.x + (long long)n * a.x_sn + (long long)g * a.D;
    double* part = a.part + 2ll * ((long long)n * a.chunks * a.C + (long long)g * a.D);
    const double rs = 1.0 / (double)a.S;
    double sum = 0.0;
    over_chunks(a, part, col, [&](int c, double p, double q) {
        sum += fma(p, rs, (double)(float)x0[c]);
        part[2ll * c] = p;
        part[2ll * c + 1] = q;
    });
    const double mean = block_sum(sum, sh) / (double)a.D;
    double m2 = 0.0;
    for (int c = threadIdx.x; c < a.D; c += blockDim.x) {   // (written by this very thread: the first walker's channels)
        const double k = (double)(float)x0[c] - mean;
        m2 = fma(k, k, fma(fma(2.0 * k, part[2ll * c], part[2ll * c + 1]), rs, m2));
    }
    const double var = block_sum(m2, sh) / (double)a.D;
    if (threadIdx.x == 0) {
        double* o = a.stats + 2ll * blockIdx.x;
        o[0] = mean;
        o[1] = 1.0 / sqrt((var < 0.0 ? 0.0 : var) + a.eps);   // (rounding may leave a constant group below 0; a NaN stays)
    }
}

// what a tile kernel keeps of its V channels
template <int V> struct Channels {
    double mean[V], rstd[V];
    float w[V], b[V];
    int group[V];
    __device__ __forceinline__ Channels(const GnArgs& a, long long n, int c0) {
        int g = c0 / a.D, r = c0 - g * a.D;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            group[k] = g;
            if (++r == a.D) {
                r = 0;
                ++g;
            }
        }
        const double* st = a.stats + 2ll * n * a.G;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            mean[k] = st[2 * group[k]];
            rstd[k] = st[2 * group[k] + 1];
        }
        load_param<V>(a.w, c0, 1.f, w);
        load_param<V>(a.b, c0, 0.f, b);
    }
};

template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnThreads) void gn_tile_apply_kernel(GnArgs a) {
    const unsigned n = blockIdx.x / (unsigned)a.chunks, ch = blockIdx.x - n * (unsigned)a.chunks;
    const Tile t = tile_of(a, a.C / V, blockIdx.y);
    if (!t.on) return;
    const Channels<V> c(a, n, t.vx * V);
    double sc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sc[k] = c.rstd[k] * (double)c.w[k];
    const float slope = a.slope;
    const T* x = (const T*)a.x + (long long)n * a.x_sn + t.vx * V;
    T* y = (T*)a.out + (long long)n * a.S * a.C + t.vx * V;
    const long long s0 = (long long)ch * a.chunk_rows, s1 = s0 + a.chunk_rows < a.S ? s0 + a.chunk_rows : a.S, xs = a.x_ss, C = a.C;
    walk<4, V>(s0 + t.ty, s1, t.rows, [&](long long s, float (&v)[V]) { load_vec<T, V>(x + s * xs, v); },
               [&](long long s, float (&v)[V]) {
#pragma unroll
                   for (int k = 0; k < V; ++k) v[k] = act_value(fma((double)v[k] - c.mean[k], sc[k], (double)c.b[k]), ACT, slope);
                   store_vec<T, V>(y + s * C, v);
               });
}

// per channel: sums of dz xh and dz over a range of rows
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnThreads) void gn_tile_bwd_sum_kernel(GnArgs a) {
    const unsigned n = blockIdx.x / (unsigned)a.chunks, ch = blockIdx.x - n * (unsigned)a.chunks;
    const Tile t = tile_of(a, a.C / V, blockIdx.y);
    double p[V], q[V];
#pragma unroll
    for (int k = 0; k < V; ++k) p[k] = q[k] = 0.0;
    if (t.on) {
        const Channels<V> c(a, n, t.vx * V);
        const float slope = a.slope;
        const T* x = (const T*)a.x + (long long)n * a.x_sn + t.vx * V;
        const T* dy = (const T*)a.dy + (long long)n * a.dy_sn + t.vx * V;
        const long long s0 = (long long)ch * a.chunk_rows, s1 = s0 + a.chunk_rows < a.S ? s0 + a.chunk_rows : a.S;
        walk<2, 2 * V>(s0 + t.ty, s1, t.rows,
                       [&](long long s, float (&v)[2 * V]) {
                           load_vec<T, V>(x + s * a.x_ss, reinterpret_cast<float(&)[V]>(v));
                           load_vec<T, V>(dy + s * a.dy_ss, reinterpret_cast<float(&)[V]>(v[V]));
                       },
                       [&](long long, float (&v)[2 * V]) {
#pragma unroll
                           for (int k = 0; k < V; ++k) {
                               const double xh = ((double)v[k] - c.mean[k]) * c.rstd[k];
                               const double dz = (double)(v[V + k] * act_slope(fma(xh, (double)c.w[k], (double)c.b[k]), ACT, slope));
                               p[k] = fma(dz, xh, p[k]);
                               q[k] += dz;
                           }
                       });
    }
    column_sum<V>(p, q, a, t);
    if (t.on && t.ty == 0)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            double* o = a.part + 2ll * ((long long)blockIdx.x * a.C + t.vx * V + k);
            o[0] = p[k];
            o[1] = q[k];
        }
}

// One workgroup per (n, g): the group's two means, and its channels' sums over the chunks on the way
__global__ __launch_bounds__(kMergeThreads) void gn_bwd_coef_kernel(GnArgs a) {
    __shared__ double sh[kMergeThreads / 64], col[kMergeThreads * 2];
    const unsigned n = blockIdx.x / (unsigned)a.G, g = blockIdx.x - n * (unsigned)a.G;
    double s1 = 0.0, s2 = 0.0;
    over_chunks(a, a.part + 2ll * ((long long)n * a.chunks * a.C + (long long)g * a.D), col, [&](int c, double p, double q) {
        const long long at = 2ll * ((long long)n * a.C + (long long)g * a.D + c);
        if (a.chan != a.part) {
            a.chan[at] = p;
            a.chan[at + 1] = q;
        }
        const double wt = a.w ? (double)a.w[(long long)g * a.D + c] : 1.0;
        s1 = fma(wt, q, s1);
        s2 = fma(wt, p, s2);
    });
    const double inv = 1.0 / ((double)a.S * a.D);
    s1 = block_sum(s1, sh) * inv;
    s2 = block_sum(s2, sh) * inv;
    if (threadIdx.x == 0) {
        a.coef[2ll * blockIdx.x] = s1;
        a.coef[2ll * blockIdx.x + 1] = s2;
    }
}

template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnThreads) void gn_tile_bwd_apply_kernel(GnArgs a) {
    const unsigned n = blockIdx.x / (unsigned)a.chunks, ch = blockIdx.x - n * (unsigned)a.chunks;
    const Tile t = tile_of(a, a.C / V, blockIdx.y);
    if (!t.on) return;
    const Channels<V> c(a, n, t.vx * V);
    float f1[V], f2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const long long u = (long long)n * a.G + c.group[k];
        f1[k] = (float)a.coef[2 * u];
        f2[k] = (float)a.coef[2 * u + 1];
    }
    const float slope = a.slope;
    const T* x = (const T*)a.x + (long long)n * a.x_sn + t.vx * V;
    const T* dy = (const T*)a.dy + (long long)n * a.dy_sn + t.vx * V;
    T* o = (T*)a.out + (long long)n * a.S * a.C + t.vx * V;
    const long long s0 = (long long)ch * a.chunk_rows, s1 = s0 + a.chunk_rows < a.S ? s0 + a.chunk_rows : a.S;
    const long long xs = a.x_ss, ds = a.dy_ss, C = a.C;
    walk<2, 2 * V>(s0 + t.ty, s1, t.rows,
                   [&](long long s, float (&v)[2 * V]) {
                       load_vec<T, V>(x + s * xs, reinterpret_cast<float(&)[V]>(v));
                       load_vec<T, V>(dy + s * ds, reinterpret_cast<float(&)[V]>(v[V]));
                   },
                   [&](long long s, float (&v)[2 * V]) {
                       float r[V];
#pragma unroll
                       for (int k = 0; k < V; ++k) {
                           const double xh = ((double)v[k] - c.mean[k]) * c.rstd[k];
                           const float wd = c.w[k] * (v[V + k] * act_slope(fma(xh, (double)c.w[k], (double)c.b[k]), ACT, slope));
                           r[k] = (float)c.rstd[k] * (wd - f1[k] - (float)xh * f2[k]);
                       }
                       store_vec<T, V>(o + s * C, r);
                   });
}

// ------------------------------------------------------------------------------------------------ resident route
// A workgroup of up to 512 threads owns all S points of one sample in a block of whole groups and keeps them in registers: one
// read, one launch.  Thread -> (vector of the row, row) as in the tile route, R rows a thread at most; a vector lies in one group
// (V divides D).  The workgroups of neighbouring blocks share cache lines: consecutive numbers go to one die.
constexpr int kResThreads = 512;

__device__ __forceinline__ unsigned by_die() {   // a permutation of the grid's numbers that gives each of the 8 dies a run of them
    const unsigned n = gridDim.x, q = n >> 3, r = n & 7, die = blockIdx.x & 7;
    return die * q + min(die, r) + (blockIdx.x >> 3);
}

struct Res {
    unsigned n, blk;
    int tx, ty, rows, x, per;   // tx: vectors a row; rows: side by side; x: this thread's vector; per: vectors a group's row
    bool on;
    __device__ __forceinline__ Res(const GnArgs& a, int V) {
        const unsigned id = by_die();
        n = id / (unsigned)a.blocks_g;
        blk = id - n * (unsigned)a.blocks_g;
        per = a.D / V;
        const int groups = min(a.res_groups, a.G - (int)blk * a.res_groups);
        tx = groups * per;
        rows = (int)blockDim.x / tx;
        ty = (int)threadIdx.x / tx;
        x = (int)threadIdx.x - ty * tx;
        on = ty < rows;
    }
};

// A vector of V elements as it lies in memory.  keep(): what has been made of it is forgotten — the compiler would rather hold the
// unpacked fp32 values from one use to the next than unpack again, and spill them.
template <typename T, int V> struct Raw {
    typedef typename Bits<V * sizeof(T)>::Type Reg;
    typedef Reg Mem __attribute__((aligned(sizeof(T))));
    typename std::conditional<sizeof(Reg) == 2, uint32_t, Reg>::type bits;
    __device__ __forceinline__ void load(const T* p) { bits = *reinterpret_cast<const Mem*>(p); }
    __device__ __forceinline__ void keep() { asm("" : "+v"(bits)); }
    __device__ __forceinline__ float at(int k) const { return (float)__builtin_bit_cast(Vec<T, V>, (Reg)bits).e[k]; }
    __device__ __forceinline__ void get(float (&v)[V]) const {
        const Vec<T, V> r = __builtin_bit_cast(Vec<T, V>, (Reg)bits);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = (float)r.e[k];
    }
};

// sums of sh[ty][x] over all rows and the `per` vectors of each group, a wave a group in turn, in a fixed order -> out[group]
__device__ __forceinline__ void group_sums(const double* sh, double* out, const Res& t) {
    __syncthreads();
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6, groups = t.tx / t.per, n = t.rows * t.per;
    for (int g = threadIdx.x >> 6; g < groups; g += waves) {
        double s = 0.0;
        for (int e = lane; e < n; e += 64) {
            const int y = e / t.per;
            s += sh[y * t.tx + g * t.per + e - y * t.per];
        }
        s = lane_sum(s, 64);
        if (lane == 0) out[g] = s;
    }
    __syncthreads();
}

template <typename T, int V, int R, int ACT>
__global__ __launch_bounds__(kResThreads) void gn_res_fwd_kernel(GnArgs a) {
    __shared__ double sh[kResThreads], sums[kResThreads];
    const Res t(a, V);
    const int c0 = ((int)t.blk * a.res_groups * t.per + t.x) * V, S = (int)a.S, g = t.x / t.per;
    const T* x = (const T*)a.x + (long long)t.n * a.x_sn + c0;
    Raw<T, V> raw[R];
    float w[V], b[V];
    double s = 0.0;
    if (t.on) {
#pragma unroll
        for (int r = 0; r < R; ++r) raw[r].load(x + (long long)min(t.ty + r * t.rows, S - 1) * a.x_ss);
        load_param<V>(a.w, c0, 1.f, w);
        load_param<V>(a.b, c0, 0.f, b);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (t.ty + r * t.rows < S) {
                float v[V];
                raw[r].get(v);
#pragma unroll
                for (int k = 0; k < V; ++k) s += (double)v[k];
            }
    }
    const double count = (double)S * a.D;
    sh[threadIdx.x] = s;
    group_sums(sh, sums, t);
    const double mean = sums[g] / count;
    s = 0.0;
    if (t.on)
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (t.ty + r * t.rows < S) {
                float v[V];
                raw[r].keep();
                raw[r].get(v);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const double d = (double)v[k] - mean;
                    s = fma(d, d, s);
                }
            }
    __syncthreads();   // (everyone has read sums)
    sh[threadIdx.x] = s;
    group_sums(sh, sums, t);
    const double rstd = 1.0 / sqrt(sums[g] / count + a.eps);
    if (!t.on) return;
    if (a.stats && t.ty == 0 && t.x == g * t.per) {
        double* o = a.stats + 2ll * ((long long)t.n * a.G + (long long)t.blk * a.res_groups + g);
        o[0] = mean;
        o[1] = rstd;
    }
    double sc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sc[k] = rstd * (double)w[k];
    T* y = (T*)a.out + (long long)t.n * S * a.C + c0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = t.ty + r * t.rows;
        if (row >= S) break;
        float v[V];
        raw[r].keep();
        raw[r].get(v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = act_value(fma((double)v[k] - mean, sc[k], (double)b[k]), ACT, a.slope);
        store_vec<T, V>(y + (long long)row * a.C, v);
    }
}

template <typename T, int V, int R, int ACT>
__global__ __launch_bounds__(kResThreads) void gn_res_bwd_kernel(GnArgs a) {
    __shared__ float sh[kResThreads * V * 2];
    __shared__ double sums[2 * kResThreads];
    const Res t(a, V);
    const int c0 = ((int)t.blk * a.res_groups * t.per + t.x) * V, S = (int)a.S, g = t.x / t.per;
    const T* x = (const T*)a.x + (long long)t.n * a.x_sn + c0;
    const T* dy = (const T*)a.dy + (long long)t.n * a.dy_sn + c0;
    Raw<T, V> rx[R];
    float dz[R][V];   // (kept: its activation's slope is most of the arithmetic, 128 x 2048 x 256 bf16 was bound by having it twice)
    float w[V], b[V];
    double mean = 0.0, rstd = 0.0, few1 = 0.0, few2 = 0.0;
    constexpr bool kFew = V * (R == 4 ? 2 : R / 2 + 1) <= kGnFew;   // D >= V, and the fewest points that give a thread R rows
    const bool few = kFew && S * a.D <= kGnFew;
    if (t.on) {
        Raw<T, V> rd[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const long long row = min(t.ty + r * t.rows, S - 1);
            rx[r].load(x + row * a.x_ss);
            rd[r].load(dy + row * a.dy_ss);
        }
        load_param<V>(a.w, c0, 1.f, w);
        load_param<V>(a.b, c0, 0.f, b);
        const double* st = a.stats + 2ll * ((long long)t.n * a.G + (long long)t.blk * a.res_groups + g);
        mean = st[0];
        rstd = st[1];
#pragma unroll
        for (int k = 0; k < V; ++k) {   // one channel's sums at a time
            const double sc = rstd * (double)w[k];
            double p = 0.0, q = 0.0;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const double d = (double)rx[r].at(k) - mean;
                const float z = rd[r].at(k) * act_slope(fma(d, sc, (double)b[k]), ACT, a.slope);
                dz[r][k] = z;
                if (t.ty + r * t.rows < S) {
                    p = fma((double)z, d, p);
                    q += (double)z;
                }
            }
            sh[((int)threadIdx.x * V + k) * 2] = (float)(p * rstd);
            sh[((int)threadIdx.x * V + k) * 2 + 1] = (float)q;
            if constexpr (kFew) {
                few1 = fma((double)w[k], q, few1);
                few2 = fma((double)w[k], p * rstd, few2);
            }
        }
    }
    if (few) {   // the threads' 64-bit sums, in the place of the groups'
        sums[threadIdx.x] = few1;
        sums[kResThreads + threadIdx.x] = few2;
    }
    // The columns' sums over the rows — a column: one of the two sums of one channel —, fp32 from each thread (2^-24 of its
    // sum, for 32 KB of LDS instead of 64 with 8 channels a thread), added in 64 bits: `parts` threads a column, then a wave a group,
    // which also has the group's two means from them.
    const int cols = t.tx * V * 2, parts = cols < (int)blockDim.x ? (int)blockDim.x / cols : 1;
    __syncthreads();
    const int part = parts > 1 ? (int)threadIdx.x / cols : 0;
    double sum = 0.0;
    if (parts > 1) {
        const int col = (int)threadIdx.x - part * cols;
        if (part < parts)
            for (int y = part; y < t.rows; y += parts) sum += (double)sh[y * cols + col];
        __syncthreads();
        if (part < parts) sh[part * cols + col] = (float)sum;
        __syncthreads();
    }
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6, groups = t.tx / t.per, n = parts > 1 ? parts : t.rows;
    int side = 1;   // channels side by side in a wave; the lanes that are left share a channel's rows
    while (side < a.D && side < 64) side *= 2;
    const int e0 = lane & (side - 1), y0 = lane / side, ystep = 64 / side;
    for (int j = threadIdx.x >> 6; j < groups; j += waves) {
        double s1 = 0.0, s2 = 0.0;
        for (int base = 0; base < a.D; base += side) {
            const int e = base + e0;
            double u = 0.0, v = 0.0;
            if (e < a.D)
                for (int y = y0; y < n; y += ystep) {
                    const float2 o = *reinterpret_cast<const float2*>(sh + y * cols + 2 * (j * a.D + e));
                    u += (double)o.x;
                    v += (double)o.y;
                }
            for (int o = side; o < 64; o *= 2) {
                u += __shfl_xor(u, o);
                v += __shfl_xor(v, o);
            }
            if (e >= a.D || y0) continue;
            const long long c = ((long long)t.blk * a.res_groups + j) * a.D + e;
            if (a.dw) {
                double* o = a.chan + 2ll * ((long long)t.n * a.C + c);
                o[0] = u;
                o[1] = v;
            }
            const double wt = a.w ? (double)a.w[c] : 1.0;
            s1 = fma(wt, v, s1);
            s2 = fma(wt, u, s2);
        }
        s1 = lane_sum(s1, 64);
        s2 = lane_sum(s2, 64);
        if (lane == 0 && !few) {
            sums[2 * j] = s1;
            sums[2 * j + 1] = s2;
        }
    }
    if (few) {   // a thread a group adds up its few threads'
        few1 = few2 = 0.0;
        if ((int)threadIdx.x < groups)
            for (int y = 0; y < min(t.rows, S); ++y)
                for (int e = 0; e < t.per; ++e) {
                    few1 += sums[y * t.tx + (int)threadIdx.x * t.per + e];
                    few2 += sums[kResThreads + y * t.tx + (int)threadIdx.x * t.per + e];
                }
        __syncthreads();
        if ((int)threadIdx.x < groups) {
            sums[2 * threadIdx.x] = few1;
            sums[2 * threadIdx.x + 1] = few2;
        }
    }
    __syncthreads();
    if (!t.on) return;
    const double s1 = sums[2 * g], s2 = sums[2 * g + 1];
    const double inv = 1.0 / ((double)S * a.D);
    T* o = (T*)a.out + (long long)t.n * S * a.C + c0;
    if constexpr (kFew)
        if (few) {
            const double m1 = s1 * inv, k2 = -rstd * (s2 * inv);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int row = t.ty + r * t.rows;
                if (row >= S) break;
                float v[V];
                rx[r].get(v);
#pragma unroll
                for (int k = 0; k < V; ++k) v[k] = grad_few((double)v[k] - mean, dz[r][k], w[k], rstd, m1, k2);
                store_vec<T, V>(o + (long long)row * a.C, v);
            }
            return;
        }
    // dx = (rstd w) dz + ((x - mean) c2 + c1), rstd w and the sum in brackets rounded to fp32 (32 x 2048 x 256 bf16 29 us, 31 with all of it
    // in 64 bits, for which there are not enough registers)
    const double c1 = -rstd * (s1 * inv), c2 = -rstd * rstd * (s2 * inv);
#pragma unroll
    for (int k = 0; k < V; ++k) w[k] *= (float)rstd;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int row = t.ty + r * t.rows;
        if (row >= S) break;
        float v[V];
        rx[r].keep();
        rx[r].get(v);
#pragma unroll
        for (int k = 0; k < V; ++k) v[k] = fmaf(w[k], dz[r][k], (float)fma((double)v[k] - mean, c2, c1));
        store_vec<T, V>(o + (long long)row * a.C, v);
    }
}

// dw, db: the sums [rows][C][2] over their rows, 32 channels and 32 row walkers per workgroup; more than one range of rows (gridDim.y):
// the ranges' sums, [range][C][2]
template <typename P>
__global__ __launch_bounds__(1024) void gn_param_grad_kernel(const P* part, long long rows, int C, float* dw, float* db, double* ranges) {
    __shared__ double sh[1024 * 2];
    const int col = threadIdx.x & 31, ty = threadIdx.x >> 5, c = (int)blockIdx.x * 32 + col;
    const long long per = (rows + gridDim.y - 1) / gridDim.y, r1 = min(rows, (blockIdx.y + 1) * per);
    double p = 0.0, q = 0.0;
    if (c < C)
#pragma unroll 8
        for (long long r = blockIdx.y * per + ty; r < r1; r += 32) {
            p += (double)part[2 * (r * C + c)];
            q += (double)part[2 * (r * C + c) + 1];
        }
    sh[2 * threadIdx.x] = p;
    sh[2 * threadIdx.x + 1] = q;
    __syncthreads();
    if (ty == 0 && c < C) {
        for (int y = 1; y < 32; ++y) {
            p += sh[2 * (y * 32 + col)];
            q += sh[2 * (y * 32 + col) + 1];
        }
        if (ranges) {
            ranges[2 * ((long long)blockIdx.y * C + c)] = p;
            ranges[2 * ((long long)blockIdx.y * C + c) + 1] = q;
        } else {
            dw[c] = (float)p;
            db[c] = (float)q;
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side
struct GnPlan {
    int V, es;            // elements per access, bytes of one
    bool unit, res;
    int res_rows, res_groups, res_blocks, res_threads;
    int items, lanes;     // unit
    int per, blocks_g, blocks_n;
    int tx, blocks_c, chunks, merge;   // merge: threads that merge a group's partial sums
    size_t part, more, ranges;         // tile: bytes of the partial sums and of the channels' sums; where gn_param_grad's begin
    long long chunk_rows;
    bool fits;                         // false: a launch would need kGnMost threads or more
};

constexpr long long kGnMost = (1ll << 32) - 1024;   // threads of a launch: below 2^32 when rounded up to whole workgroups

int elem_bytes(int dtype) { return dtype == DGG_F32 ? 4 : 2; }

// The widest access, of at most 16 bytes, that divides a range of channels (256 x 256 x 34 bf16 in 17 groups with two elements instead
// of one: 11.6 -> 9.3 us forward, 18.6 -> 15.1 backward); `fits`: that is no wider than it.  For rows the unit route lets a group's last
// vector overlap the one before it: 4096 x 515 bf16 in 5 groups 13.8 -> 7.7 us forward, 22.4 -> 17.2 backward, 20000 x 105 f32 in 7 17.1
// -> 8.8 and 22.6 -> 15.3; elsewhere the masks cost more than the accesses (64 x 4096 x 33 bf16 in 11, tile: 27 us element by element, 44
// with overlapping vectors; 3000 x 9 x 33 in 11, unit: 11 and 15).
int gn_width(int dtype, int width, bool fits) {
    const int W = 16 / elem_bytes(dtype);
    for (int V = W; V > 1; V /= 2)
        if (fits ? width >= V : width % V == 0) return V;
    return 1;
}

void gn_tile_plan(GnPlan& P, long long N, long long S, int C) {
    const int vecs = C / P.V;
    P.blocks_c = (vecs + kGnThreads - 1) / kGnThreads;
    P.tx = (vecs + P.blocks_c - 1) / P.blocks_c;
    // about 1024 workgroups (2048: 9 x 61743 x 16 bf16 35 instead of 26 us forward), of at least 64 rows each and two for every thread
    // (the partial sums stay small beside the data), or about 512 of at least 8 and two (2 x 269 x 666 f16 in 18 groups, forward and
    // backward: 46 -> 28 us)
    const long long rows = 2 * (kGnThreads / P.tx), least = rows > 64 ? rows : 64, few = rows > 8 ? rows : 8;
    long long want = 1024 / (N * P.blocks_c), less = 512 / (N * P.blocks_c);
    if (want > (S + least - 1) / least) want = (S + least - 1) / least;
    if (less > (S + few - 1) / few) less = (S + few - 1) / few;
    if (want < less) want = less;
    if (want < 1) want = 1;
    P.chunk_rows = (S + want - 1) / want;
    P.chunks = (int)((S + P.chunk_rows - 1) / P.chunk_rows);
}

// A group in the registers of a part of a wave, 4 vectors a lane at most (points backward: one), or, rows, of a workgroup, 32 elements a thread
// at most (8192 x 4096 bf16 in one group: 107 us forward and 754 backward with 8 vectors a lane of a wave, which spills, 62 and 78 so).
bool gn_unit_plan(GnPlan& P, long long S, int D, bool backward) {
    const long long nv = S * (long long)vectors(D, P.V), most = S == 1 ? 256ll * (32 / P.V > 8 ? 8 : 32 / P.V) : backward ? 64 : 256;
    if (S > most || nv > most) return false;
    P.lanes = 1;
    if (nv > 256) P.lanes = kGnThreads;
    else while (P.lanes < 64 && P.lanes < nv) P.lanes *= 2;
    P.items = 1;
    while (P.items * P.lanes < nv) P.items *= 2;
    return true;
}

// Resident: whole samples in registers, 16 vectors a thread (backward: of x and of dy) and 512 threads at most.  Resident against
// tile, forward / backward, us: 32 x 2048 x 256 bf16 in 32 groups 21 / 29 against 29 / 47, 128 x 2048 x 256 69 / 128 against 102 / 190,
// 5 x 1237 x 132 f16 in 11 8.5 / 12.2 against 13.4 / 16.5, 4 x 4096 x 64 f32 in 8 10.8 / 14.5 against 12.2 / 15.2.
bool gn_res_plan(GnPlan& P, long long N, long long S, int C, int G) {
    if (S > 16 * kResThreads) return false;
    const int per = C / G / P.V;
    if (per > kResThreads) return false;
    // as many groups side by side as leave every thread 16 rows ..
    int groups = (int)(16ll * kResThreads / (S * per));
    if (groups > kResThreads / per) groups = kResThreads / per;
    while (groups > 0 && (long long)(kResThreads / (groups * per)) * 16 < S) --groups;
    if (groups < 1) return false;
    if (groups > G) groups = G;
    // .. but 256 workgroups at least, down to 64 bytes of a row each (and 64 workgroups whatever it takes; 128 or 512, and 32 or 128
    // bytes, make 3 % at most either way, 64 x 64 x 64 bf16 backward excepted: 7.8, 8.2 and 9.2 us with 32, 64 and 128 bytes)
    const int line = 64 / (P.V * P.es);
    while (groups > 1 && N * ((G + groups - 1) / groups) < 256 && ((groups / 2) * per >= line || N * ((G + groups - 1) / groups) < 64))
        groups /= 2;
    P.res_groups = groups;
    P.res_blocks = (G + groups - 1) / groups;
    const int tx = groups * per;
    long long rows = kResThreads / tx;
    if (rows > S) rows = S;
    P.res_threads = (int)((rows * tx + 63) / 64 * 64);
    if (P.res_threads > kResThreads) P.res_threads = kResThreads;
    rows = P.res_threads / tx;
    const long long most = (S + rows - 1) / rows;
    P.res_rows = most <= 4 ? 4 : most <= 8 ? 8 : 16;
    return (long long)P.res_blocks * P.res_threads < kGnMost;   // (of one sample: gn_launches)
}

void gn_unit_bwd_grid(GnPlan& P, long long N, int G) {
    const int slots = kGnThreads / P.lanes;
    P.per = G < slots ? slots / G : 1;
    P.blocks_g = G < slots ? 1 : (G + slots - 1) / slots;
    // (16384 x 512 f32 in 32 groups, backward: 54, 37, 30 us with 256, 512, 1024 workgroups)
    long long nb = (N + P.per - 1) / P.per, most = 1024 / P.blocks_g;
    if (most < 1) most = 1;
    P.blocks_n = (int)(nb < most ? nb : most);
}

// Ranges of rows in the sum that makes dw and db (resident and tile: a row a sample; the unit route has 1024 at most): one where the launch
// is a latency or two long, else of 512 rows or more (20000 x 100 x 16 bf16 in 2 groups: the backward pass takes 166 us in all, 231 with one
// range; 4096 x 100 x 64 in 4 77 and 90)
int gn_ranges(long long rows) { return rows <= 1024 ? 1 : rows < 64 * 512 ? (int)((rows + 511) / 512) : 64; }

int gn_check(long long N, long long S, int C, int G, int act, int dtype, const char* who) {
    if (N < 1 || S < 1 || C < 1 || G < 1 || C % G != 0) {
        set_error_text("%s: N, S, C, groups must be positive and groups must divide C (N = %lld, S = %lld, C = %d, groups = %d)",
                       who, N, S, C, G);
        return DGG_ERR_INVALID;
    }
    if (dtype < DGG_F32 || dtype > DGG_F16 || act < DGG_ACT_NONE || act > DGG_ACT_SILU) {
        set_error_text("%s: unknown type %d or activation %d", who, dtype, act);
        return DGG_ERR_INVALID;
    }
    // 32-bit workgroup and unit numbers; element offsets are 64 bits wide
    if (N > 0x7fffffffll / G || S > 0x7fffffffll || C > (1 << 24)) {
        set_error_text("%s: N * groups and S must stay below 2^31, C up to 2^24 (N = %lld, S = %lld, C = %d)", who, N, S, C);
        return DGG_ERR_INVALID;
    }
    return DGG_OK;
}

// The route of a call, its launches and the workspace it needs (part and more: see gn_run).
size_t gn_plan(GnPlan& P, long long N, long long S, int C, int G, int dtype, bool backward, bool grads) {
    const int D = C / G;
    P.es = elem_bytes(dtype);
    P.V = gn_width(dtype, D, S == 1);
    P.unit = gn_unit_plan(P, S, D, backward);
    if (!P.unit) P.V = gn_width(dtype, D, false);
    P.res = (S > 1 || !P.unit) && gn_res_plan(P, N, S, C, G);
    // Points that fit both go to the units unless those take 1.5 times the resident route's threads (a lane with a vector costs 8 ns a
    // thousand, a thread with its rows 12 to 17), backward where there are samples for every slot too.  Unit against resident, us, forward:
    // 20000 x 2 x 16 bf16 in 2 groups 3.8 / 26, 4000 x 16 x 32 f32 in 4 8.0 / 11.5, 3000 x 9 x 33 bf16 in 11 11 / 19, 300 x 37 x 15 f32 in 5
    // 4.5 / 5.4, 64 x 100 x 15 in 5 6.0 / 4.6, 1779 x 6 x 459 bf16 in 51 50 / 37, 256 x 256 x 128 in 8 30 / 15; backward: 20000 x 2 x 16 14 /
    // 123, 4096 x 4 x 256 in 32 20 / 92, 4000 x 16 x 32 19 / 29, 64 x 64 x 64 in 8 12.4 / 9.3; rows 1024 x 512 f32 in 32 4.3 / 16.9 and 9.7 /
    // 26.4.
    if (P.unit && P.res) {
        const long long lanes = N * G * P.lanes * P.items, threads = N * P.res_blocks * P.res_threads;
        P.unit = 2 * lanes <= 3 * threads && !(backward && N * P.res_blocks < 512);
        P.res = !P.unit;
    }
    P.part = P.more = 0;
    P.fits = true;
    size_t need = 0;
    if (P.unit) {
        if (backward) gn_unit_bwd_grid(P, N, G);
        need = grads ? (size_t)P.blocks_n * C * 2 * sizeof(float) : 0;
    } else if (P.res) {
        need = grads ? (size_t)N * C * 2 * sizeof(double) : 0;
    } else {
        P.V = gn_width(dtype, C, false);
        gn_tile_plan(P, N, S, C);
        P.merge = (long long)P.chunks * D > 1024 ? kMergeThreads : kGnThreads;
        P.fits = N * P.chunks * kGnThreads < kGnMost && N * G * P.merge < kGnMost && P.blocks_c <= 65535;
        const size_t chan = (size_t)N * C * 2 * sizeof(double);
        P.part = chan * P.chunks;
        P.more = backward && P.chunks > 1 ? chan : 0;
        need = P.part + P.more + (size_t)N * G * 2 * sizeof(double);
    }
    P.ranges = need;   // where gn_param_grad's partial sums begin
    return need + (grads && !P.unit && gn_ranges(N) > 1 ? (size_t)gn_ranges(N) * C * 2 * sizeof(double) : 0);
}

template <typename P> void gn_param_grad(const GnArgs& a, const P* part, long long rows, hipStream_t st) {
    const int ranges = gn_ranges(rows);
    const dim3 grid((unsigned)((a.C + 31) / 32), ranges), block(1024);
    hipLaunchKernelGGL((gn_param_grad_kernel<P>), grid, block, 0, st, part, rows, a.C, a.dw, a.db, ranges > 1 ? a.ranges : nullptr);
    if (ranges > 1)
        hipLaunchKernelGGL((gn_param_grad_kernel<double>), dim3(grid.x), block, 0, st, (const double*)a.ranges, (long long)ranges, a.C, a.dw,
                           a.db, (double*)nullptr);
}

// launch(samples of a call): all of them, or, where they need `threads` each and kGnMost together, ranges of them in turn
template <typename Launch> void gn_launches(const GnArgs& a, long long threads, int es, Launch launch) {
    const long long most = kGnMost / threads;
    if (a.N <= most) return launch(a);
    for (long long n = 0; n < a.N; n += most) {
        GnArgs r = a;
        r.N = a.N - n < most ? a.N - n : most;
        r.x = (const char*)a.x + n * a.x_sn * es;
        r.dy = a.dy ? (const char*)a.dy + n * a.dy_sn * es : nullptr;
        r.out = (char*)a.out + n * a.S * a.C * es;
        r.stats = a.stats ? a.stats + 2 * n * a.G : nullptr;
        r.chan = a.dw ? a.chan + 2 * n * a.C : nullptr;
        launch(r);
    }
}

#define GN_ACT(act, kernel, grid)                                                                                       \
    if (act == DGG_ACT_LEAKY_RELU) hipLaunchKernelGGL((kernel<T, V, DGG_ACT_LEAKY_RELU>), grid, block, 0, st, a);       \
    else if (act == DGG_ACT_SILU) hipLaunchKernelGGL((kernel<T, V, DGG_ACT_SILU>), grid, block, 0, st, a);              \
    else hipLaunchKernelGGL((kernel<T, V, DGG_ACT_NONE>), grid, block, 0, st, a);

// items: 1, 2, 4 vectors a lane of a wave (MANY: more than 1 only there); 2, 4, 8 (16 bits: 4) widest ones a thread of a workgroup
#define GN_UNIT_I(kernel, EVEN, MANY, ...)                                                                                    \
    if (P.lanes == kGnThreads) {                                                                                              \
        if constexpr (V == 16 / (int)sizeof(T)) {                                                                             \
            if (P.items == 2) hipLaunchKernelGGL((kernel<T, V, EVEN, 2, true __VA_ARGS__>), grid, block, 0, st, a);            \
            else if (P.items == 4 || V == 8) hipLaunchKernelGGL((kernel<T, V, EVEN, 4, true __VA_ARGS__>), grid, block, 0, st, a); \
            else hipLaunchKernelGGL((kernel<T, V, EVEN, V == 8 ? 4 : 8, true __VA_ARGS__>), grid, block, 0, st, a);            \
        }                                                                                                                     \
    } else if constexpr (MANY) {                                                                                              \
        if (P.items == 1) hipLaunchKernelGGL((kernel<T, V, EVEN, 1, false __VA_ARGS__>), grid, block, 0, st, a);               \
        else if (P.items == 2) hipLaunchKernelGGL((kernel<T, V, EVEN, 2, false __VA_ARGS__>), grid, block, 0, st, a);          \
        else hipLaunchKernelGGL((kernel<T, V, EVEN, 4, false __VA_ARGS__>), grid, block, 0, st, a);                            \
    } else hipLaunchKernelGGL((kernel<T, V, EVEN, 1, false __VA_ARGS__>), grid, block, 0, st, a);
#define GN_COMMA ,
// POINTS: S > 1 may come here, whose accesses divide the channels.  Rows have narrow accesses only where a group is narrower than a wide one:
// two vectors, in two lanes
#define GN_UNIT(kernel, POINTS, ...)                                                                                          \
    constexpr bool widest = V == 16 / (int)sizeof(T);                                                                         \
    if (V == 1 || a.D % V == 0) { GN_UNIT_I(kernel, true, widest || POINTS, __VA_ARGS__) }                                    \
    else { GN_UNIT_I(kernel, (V == 1), widest || (V == 1 && POINTS), __VA_ARGS__) }

#define GN_RES(act, kernel, R)                                                                                             \
    if (act == DGG_ACT_LEAKY_RELU) hipLaunchKernelGGL((kernel<T, V, R, DGG_ACT_LEAKY_RELU>), grid, block, 0, st, a);       \
    else if (act == DGG_ACT_SILU) hipLaunchKernelGGL((kernel<T, V, R, DGG_ACT_SILU>), grid, block, 0, st, a);              \
    else hipLaunchKernelGGL((kernel<T, V, R, DGG_ACT_NONE>), grid, block, 0, st, a);

template <typename T, int V> int gn_forward_v(const GnPlan& P, GnArgs& a, hipStream_t st) {
    if (P.unit) {
        gn_launches(a, (long long)a.G * P.lanes, sizeof(T), [&](const GnArgs& a) {
            const dim3 grid((unsigned)((a.N * a.G * P.lanes + kGnThreads - 1) / kGnThreads)), block(kGnThreads);
            GN_UNIT(gn_unit_fwd_kernel, true, )
        });
        return check_launch("group_norm forward");
    }
    if (P.res) {
        gn_launches(a, (long long)P.res_blocks * P.res_threads, sizeof(T), [&](const GnArgs& a) {
            const dim3 grid((unsigned)(a.N * P.res_blocks)), block(P.res_threads);
            if (P.res_rows == 4) { GN_RES(a.act, gn_res_fwd_kernel, 4) }
            else if (P.res_rows == 8) { GN_RES(a.act, gn_res_fwd_kernel, 8) }
            else { GN_RES(a.act, gn_res_fwd_kernel, 16) }
        });
        return check_launch("group_norm forward");
    }
    const dim3 grid((unsigned)(a.N * P.chunks), P.blocks_c), block(kGnThreads);
    hipLaunchKernelGGL((gn_tile_sum_kernel<T, V>), grid, block, 0, st, a);
    hipLaunchKernelGGL((gn_stats_kernel<T>), dim3((unsigned)(a.N * a.G)), dim3(P.merge), 0, st, a);
    GN_ACT(a.act, gn_tile_apply_kernel, grid)
    return check_launch("group_norm forward");
}

template <typename T, int V> int gn_backward_v(const GnPlan& P, GnArgs& a, hipStream_t st) {
    const dim3 block(kGnThreads);
    if (P.unit) {
        if (!a.dw) a.part = nullptr;
        const dim3 grid((unsigned)P.blocks_g * P.blocks_n);
        if (a.S == 1) { GN_UNIT(gn_unit_bwd_kernel, false, GN_COMMA false) }
        else hipLaunchKernelGGL((gn_unit_bwd_kernel<T, V, true, 1, false, true>), grid, block, 0, st, a);
        if (a.dw) gn_param_grad(a, (const float*)a.part, P.blocks_n, st);
        return check_launch("group_norm backward");
    }
    if (P.res) {
        gn_launches(a, (long long)P.res_blocks * P.res_threads, sizeof(T), [&](const GnArgs& a) {
            const dim3 grid((unsigned)(a.N * P.res_blocks)), block(P.res_threads);
            if (P.res_rows == 4) { GN_RES(a.act, gn_res_bwd_kernel, 4) }
            else if (P.res_rows == 8) { GN_RES(a.act, gn_res_bwd_kernel, 8) }
            else { GN_RES(a.act, gn_res_bwd_kernel, 16) }
        });
        if (a.dw) gn_param_grad(a, (const double*)a.chan, a.N, st);
        return check_launch("group_norm backward");
    }
    const dim3 grid((unsigned)(a.N * P.chunks), P.blocks_c);
    GN_ACT(a.act, gn_tile_bwd_sum_kernel, grid)
    hipLaunchKernelGGL(gn_bwd_coef_kernel, dim3((unsigned)(a.N * a.G)), dim3(P.merge), 0, st, a);
    if (a.dw) gn_param_grad(a, (const double*)a.chan, a.N, st);
    GN_ACT(a.act, gn_tile_bwd_apply_kernel, grid)
    return check_launch("group_norm backward");
}

template <typename T> int gn_dispatch(bool backward, const GnPlan& P, GnArgs& a, hipStream_t st) {
    constexpr int W = 16 / sizeof(T);
    if (P.V == W) return backward ? gn_backward_v<T, W>(P, a, st) : gn_forward_v<T, W>(P, a, st);
    if (W > 4 && P.V == 4) return backward ? gn_backward_v<T, 4>(P, a, st) : gn_forward_v<T, 4>(P, a, st);
    if (P.V == 2) return backward ? gn_backward_v<T, 2>(P, a, st) : gn_forward_v<T, 2>(P, a, st);
    return backward ? gn_backward_v<T, 1>(P, a, st) : gn_forward_v<T, 1>(P, a, st);
}

int gn_refuse(long long N, long long S, int C, int G, const char* who) {
    set_error_text("%s: %lld samples of %lld points of %d channels in %d groups need a launch of 2^32 threads or of more than 65535 blocks of "
                   "channels", who, N, S, C, G);
    return DGG_ERR_INVALID;
}

int gn_run(bool backward, GnArgs& a, int dtype, void* ws, size_t ws_bytes, hipStream_t st, const char* who) {
    a.D = a.C / a.G;
    GnPlan P = {};
    const size_t need = gn_plan(P, a.N, a.S, a.C, a.G, dtype, backward, backward && a.dw);
    if (!P.fits) return gn_refuse(a.N, a.S, a.C, a.G, who);
    if (need && (!ws || ws_bytes < need || (uintptr_t)ws % 8)) {
        set_error_text("%s: the workspace has %zu bytes, %zu (8-byte aligned) are needed", who, ws_bytes, need);
        return DGG_ERR_WORKSPACE;
    }
    const int es = elem_bytes(dtype);
    if ((uintptr_t)a.x % es || (uintptr_t)a.out % es || (uintptr_t)a.dy % es) {
        set_error_text("%s: a tensor that does not begin at an element's address", who);
        return DGG_ERR_INVALID;
    }
    a.chan = (double*)ws;
    if (P.unit) {
        a.lanes = P.lanes;
        a.blocks_g = P.blocks_g;
        a.blocks_n = P.blocks_n;
    } else if (P.res) {
        a.res_groups = P.res_groups;
        a.blocks_g = P.res_blocks;
    } else {
        a.chunks = P.chunks;
        a.chunk_rows = P.chunk_rows;
        a.tx = P.tx;
        a.chan = (double*)((char*)ws + (P.more ? P.part : 0));
        a.coef = (double*)((char*)ws + P.part + P.more);
        if (!a.stats) a.stats = a.coef;   // a forward without a backward keeps its statistics in the workspace
    }
    a.ranges = (double*)((char*)ws + P.ranges);
    a.part = (double*)ws;
    return dtype == DGG_F32 ? gn_dispatch<float>(backward, P, a, st)
         : dtype == DGG_BF16 ? gn_dispatch<__bf16>(backward, P, a, st) : gn_dispatch<_Float16>(backward, P, a, st);
}

}  // namespace
}  // namespace dgg

using namespace dgg;

extern "C" {

int64_t dgg_group_norm_workspace_bytes(int64_t N, int64_t S, int C, int groups, int dtype, int backward) {
    const int rc = gn_check(N, S, C, groups, DGG_ACT_NONE, dtype, "dgg_group_norm_workspace_bytes");
    if (rc != DGG_OK) return rc;
    GnPlan P = {};
    const size_t need = gn_plan(P, N, S, C, groups, dtype, backward != 0, backward != 0);
    return P.fits ? (int64_t)need : gn_refuse(N, S, C, groups, "dgg_group_norm_workspace_bytes");
}

int dgg_group_norm_act_forward(const void* x, int64_t x_stride_n, int64_t x_stride_s, int64_t N, int64_t S, int C, int groups,
                               const float* weight, const float* bias, double eps, int act, float slope, int dtype, void* y,
                               double* stats, void* ws, size_t ws_bytes, void* stream) {
    const char* who = "dgg_group_norm_act_forward";
    const int rc = gn_check(N, S, C, groups, act, dtype, who);
    if (rc != DGG_OK) return rc;
    if (!x || !y || x_stride_n < 0 || x_stride_s < 0 || !(eps >= 0.0)) {
        set_error_text("%s: x, y, strides >= 0 and eps >= 0 are needed", who);
        return DGG_ERR_INVALID;
    }
    GnArgs a = {};
    a.x = x; a.out = y; a.w = weight; a.b = bias; a.stats = stats;
    a.x_sn = x_stride_n; a.x_ss = x_stride_s;
    a.N = N; a.S = S; a.C = C; a.G = groups;
    a.act = act; a.slope = slope; a.eps = eps;
    return gn_run(false, a, dtype, ws, ws_bytes, (hipStream_t)stream, who);
}

int dgg_group_norm_act_backward(const void* dy, int64_t dy_stride_n, int64_t dy_stride_s, const void* x, int64_t x_stride_n,
                                int64_t x_stride_s, int64_t N, int64_t S, int C, int groups, const float* weight,
                                const float* bias, int act, float slope, int dtype, const double* stats, void* dx,
                                float* dweight, float* dbias, void* ws, size_t ws_bytes, void* stream) {
    const char* who = "dgg_group_norm_act_backward";
    const int rc = gn_check(N, S, C, groups, act, dtype, who);
    if (rc != DGG_OK) return rc;
    if (!dy || !x || !stats || !dx || x_stride_n < 0 || x_stride_s < 0 || dy_stride_n < 0 || dy_stride_s < 0 || !dweight != !dbias) {
        set_error_text("%s: dy, x, stats, dx, strides >= 0, and both or none of dweight and dbias are needed", who);
        return DGG_ERR_INVALID;
    }
    GnArgs a = {};
    a.dy = dy; a.x = x; a.out = dx; a.w = weight; a.b = bias; a.stats = const_cast<double*>(stats);
    a.dy_sn = dy_stride_n; a.dy_ss = dy_stride_s; a.x_sn = x_stride_n; a.x_ss = x_stride_s;
    a.N = N; a.S = S; a.C = C; a.G = groups;
    a.act = act; a.slope = slope; a.dw = dweight; a.db = dbias;
    return gn_run(true, a, dtype, ws, ws_bytes, (hipStream_t)stream, who);
}

}  // extern "C"
