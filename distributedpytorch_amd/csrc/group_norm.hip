// Group normalisation of a channels-last map, fused with a residual and an activation, forward and backward.
//
//   per image n and group g over the m = (C / G) H W elements of the group
//     mean, var = E[x], E[(x - mean)^2]          rstd = 1 / sqrt(var + eps)        xhat = (x - mean) rstd
//     z = w_c xhat + b_c (+ residual)            y = act(z),   act: identity, ReLU, SiLU z / (1 + e^-z)
//   backward, dz = dy act'(z)
//     db_c = sum dz      dw_c = sum dz xhat      m1 = E[w dz]      m2 = E[w dz xhat]      (E over the group)
//     dx = rstd (w dz - m1 - xhat m2)            d residual = dz
//
// Bound by memory: about 10 (forward) to 25 (backward) operations an element against 4 to 8 bytes.  Sums run over whole
// groups before the first output exists, so the map is read twice: statistics, a small kernel that joins the row splits,
// and the element pass.
//
// Measured on 16 x 256 x 129 x 129, bf16, SiLU, 32 groups (a map of 136 MB; a copy of 2 GiB moves 4.9 TB/s):
//   gn_stats 38 us (3.6 TB/s)   gn_finish 6   gn_apply 54 (5.1)   gn_bwd_reduce 61 (4.4)   gn_bwd_join 7   gn_bwd_apply 81 (5.1)
//
// Precision.  Statistics are sums of differences from a per-channel pivot (the mean of four spread positions), so a map
// whose mean is far larger than its spread loses nothing to cancellation; channels are joined by their means and their
// squared deviations (all terms positive) in 64 bits.  z is formed as x a + b, for ReLU with a and b split into a rounded value
// and its remainder: its error is relative to z itself, so ReLU's border falls where the definition puts it (before a residual
// is added: the sum's error is relative to the larger term).
// No atomics: every sum has one order.
#include "common.h"

namespace {

enum Act { kNone = 0, kRelu = 1, kSilu = 2 };

typedef _Float16 f16;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<bf16_raw>(bf16_raw v) { return bf2f(v); }
template <> __device__ __forceinline__ float to_f<f16>(f16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_raw from_f<bf16_raw>(float v) { return f2bf(v); }
template <> __device__ __forceinline__ f16 from_f<f16>(float v) { return (f16)v; }

// V elements of 16 bytes in all (V > 1) or a single one
template <typename T, int V> struct Pack {
    uint4 raw;
    __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ float get(int i) const {
        const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (__is_same(T, bf16_raw)) return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
        else return (float)__builtin_bit_cast(f16, (unsigned short)(w[i >> 1] >> (i & 1 ? 16 : 0)));
    }
    static __device__ __forceinline__ void store(T* p, const float* f) {
        T t[V];
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = from_f<T>(f[i]);
        uint4 u;
        __builtin_memcpy(&u, t, 16);
        *reinterpret_cast<uint4*>(p) = u;
    }
};
template <typename T> struct Pack<T, 1> {
    T one;
    __device__ __forceinline__ void load(const T* p) { one = *p; }
    __device__ __forceinline__ float get(int) const { return to_f(one); }
    static __device__ __forceinline__ void store(T* p, const float* f) { *p = from_f<T>(f[0]); }
};

// A block of 256 threads: cb neighbouring packs of a row by rpp rows; a thread keeps its channels and walks down rows.
struct Geo {
    long hw;                 // rows of an image
    int C, G, cpg;           // channels, groups, channels of a group
    int cv, cb, rpp;         // packs of a row, packs and rows of a block
    int cblocks, splits;     // blocks along a row, row ranges of an image
    long rows;               // rows of a range
    long ldx, ldr, ldd;      // elements between rows of x, the residual and dy (outputs are dense)
    float eps;
};

struct Place { long n, row, row_end; int chunk, split, lane_row; bool on; };

__device__ __forceinline__ Place place(const Geo& g, long id) {
    Place p;
    p.split = (int)(id % g.splits);
    const long t = id / g.splits;
    const int cblk = (int)(t % g.cblocks);
    p.n = t / g.cblocks;
    p.lane_row = threadIdx.x / g.cb;
    p.chunk = cblk * g.cb + (int)threadIdx.x % g.cb;
    p.on = p.lane_row < g.rpp && p.chunk < g.cv;
    p.row = p.split * g.rows + p.lane_row;
    p.row_end = (p.split + 1) * g.rows < g.hw ? (p.split + 1) * g.rows : g.hw;
    return p;
}

// sum of acc[0..K) over the `rows` lines of `cols` threads of a block of N; the result is left with the first line
template <int K, int N> __device__ __forceinline__ void join_rows(float* acc, float* lds, int cols, int rows, int line) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int k = 0; k < K; ++k) lds[k * N + tid] = acc[k];
    int s = 1;
    while (s < rows) s <<= 1;
    for (s >>= 1; s > 0; s >>= 1) {
        __syncthreads();
        if (line < s && line + s < rows)
#pragma unroll
            for (int k = 0; k < K; ++k) lds[k * N + tid] += lds[k * N + tid + s * cols];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) acc[k] = lds[k * N + tid];
}

constexpr int kUnroll = 4;   // packs in flight per thread and operand

// body(u, row) for the thread's rows: fetch(u, row) of kUnroll rows first, so that their loads are in flight together
template <typename F, typename B> __device__ __forceinline__ void walk(const Geo& g, const Place& p, F fetch, B body) {
    long r = p.row;
    const long step = g.rpp;
    for (; r + (kUnroll - 1) * step < p.row_end; r += kUnroll * step) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) fetch(u, r + u * step);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) body(u, r + u * step);
    }
    for (; r < p.row_end; r += step) { fetch(0, r); body(0, r); }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void gn_stats_kernel(Geo g, const T* __restrict__ x, float* __restrict__ part,
                                                       float* __restrict__ pivot) {
    __shared__ float lds[2 * V * 256];
    const Place p = place(g, blockIdx.x);
    float acc[2 * V];
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) acc[k] = 0.f;
    if (p.on) {
        const T* base = x + p.n * g.hw * g.ldx + (long)p.chunk * V;
        float pv[V];
#pragma unroll
        for (int i = 0; i < V; ++i) pv[i] = 0.f;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            Pack<T, V> a;
            a.load(base + (g.hw * s / 4) * g.ldx);
#pragma unroll
            for (int i = 0; i < V; ++i) pv[i] += 0.25f * a.get(i);
        }
        if (p.split == 0 && p.lane_row == 0)
#pragma unroll
            for (int i = 0; i < V; ++i) pivot[p.n * g.C + (long)p.chunk * V + i] = pv[i];
        Pack<T, V> a[kUnroll];
        walk(g, p, [&](int u, long r) { a[u].load(base + r * g.ldx); },
             [&](int u, long) {
#pragma unroll
                 for (int i = 0; i < V; ++i) {
                     const float d = a[u].get(i) - pv[i];
                     acc[i] += d;
                     acc[V + i] = fmaf(d, d, acc[V + i]);
                 }
             });
    }
    join_rows<2 * V, 256>(acc, lds, g.cb, g.rpp, p.lane_row);
    if (p.on && p.lane_row == 0) {
        float* o = part + ((p.n * g.splits + p.split) * 2) * g.C + (long)p.chunk * V;
#pragma unroll
        for (int i = 0; i < V; ++i) { o[i] = acc[i]; o[g.C + i] = acc[V + i]; }
    }
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// A team of 16, 64 or 256 threads, whole in one block of N, takes one (image, group): its items are the group's (row range,
// channel) pairs, in memory order.
struct Team { long gi, n; int c0, items, first, step; bool on; };

template <int N> __device__ __forceinline__ Team team_of(const Geo& g, long groups, int team, long block) {
    const int tid = threadIdx.x;
    Team t;
    t.step = team;
    t.gi = block * (N / team) + tid / team;
    t.on = t.gi < groups;
    t.n = t.on ? t.gi / g.G : 0;
    t.c0 = t.on ? (int)(t.gi % g.G) * g.cpg : 0;
    t.items = t.on ? g.cpg * g.splits : 0;
    t.first = tid % t.step;
    return t;
}

__device__ __forceinline__ double team_sum(double v, int team, double* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        if (o < team) v += __shfl_xor(v, o, 64);
    if (team <= 64) return v;
    const int w = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[w] = v;
    __syncthreads();
    const double* own = lds + (w & ~3);
    return (own[0] + own[1]) + (own[2] + own[3]);
}

// 1 / std.  In a group of one element xhat is zero and dx = 0 whatever the element: with 1 / std = 0 both are, where the
// difference of w dz and its mean, which is its rounding, times 1 / sqrt(eps) would not be.
__device__ __forceinline__ double inv_std(const Geo& g, double var) {
    return g.hw * g.cpg == 1 ? 0.0 : 1.0 / sqrt(var + (double)g.eps);
}

// stats[n, g] = (mean, rstd).  Every item is a sample with a mean and squared deviations of its own; all the terms that
// join them are positive.
__global__ __launch_bounds__(256) void gn_finish_kernel(Geo g, long groups, int team, const float* __restrict__ part,
                                                        const float* __restrict__ pivot, double* __restrict__ stats) {
    __shared__ double lds[4];
    const Team t = team_of<256>(g, groups, team, blockIdx.x);
    const float* base = part + t.n * g.splits * 2 * g.C + t.c0;
    const float* pv = pivot + t.n * g.C + t.c0;
    double sm = 0.0;
#pragma unroll 4
    for (int i = t.first; i < t.items; i += t.step) {
        const int s = i / g.cpg, c = i - s * g.cpg;
        const long rows = (s + 1) * g.rows < g.hw ? g.rows : g.hw - s * g.rows;
        sm += (double)rows * (double)pv[c] + (double)base[(long)s * 2 * g.C + c];
    }
    const double count = (double)g.hw * g.cpg;
    const double mean = team_sum(sm, team, lds) / count;
    double m2 = 0.0;
#pragma unroll 4
    for (int i = t.first; i < t.items; i += t.step) {
        const int s = i / g.cpg, c = i - s * g.cpg;
        const double rows = (double)((s + 1) * g.rows < g.hw ? g.rows : g.hw - s * g.rows);
        const double s1 = (double)base[(long)s * 2 * g.C + c], s2 = (double)base[(long)s * 2 * g.C + g.C + c];
        const double own = s2 - s1 * s1 / rows, d = (double)pv[c] + s1 / rows - mean;
        m2 += (own < 0.0 ? 0.0 : own) + d * d * rows;                                   // (a NaN stays one)
    }
    m2 = team_sum(m2, team, lds);
    if (t.on && t.first == 0) {
        stats[2 * t.gi] = mean;
        stats[2 * t.gi + 1] = inv_std(g, m2 / count);
    }
}

// Constants of one thread's V channels; S: how many groups its pack can touch (1: cpg is a multiple of V, else V).
template <int V, int S> struct Norm { float mh[S], ml[S], rs[S]; double mean[S], rstd[S]; };   // xhat = (x - mean) rstd

template <int V, int S>
__device__ __forceinline__ Norm<V, S> norm_of(const Geo& g, const Place& p, const double* stats) {
    Norm<V, S> c;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const double* st = stats + 2 * (p.n * g.G + (p.chunk * V + i) / g.cpg);
        c.mean[i] = st[0]; c.rstd[i] = st[1];
        c.mh[i] = (float)st[0]; c.ml[i] = (float)(st[0] - (double)c.mh[i]); c.rs[i] = (float)st[1];
    }
    return c;
}

// z from x or from d = x - mh.  With ReLU the sign of z decides whole gradients: there z = x a + b with a and b split
// into a rounded value and its remainder (near z = 0 the first product leaves z almost exactly, and the second adds what
// the rounded coefficients left out).  Elsewhere z = d a + b', whose error is a few 2^-24 of |d a| and |b'|.
template <int V, bool SPLIT> struct Coef {
    float ah[V], bh[V], al[SPLIT ? V : 1], bl[SPLIT ? V : 1];
    template <int S>
    __device__ __forceinline__ void set(int i, const Norm<V, S>& n, float w, float b) {
        const double a = (double)w * n.rstd[i % S];
        ah[i] = (float)a;
        if constexpr (SPLIT) {
            const double bb = (double)b - n.mean[i % S] * a;
            bh[i] = (float)bb;
            al[i] = (float)(a - (double)ah[i]);
            bl[i] = (float)(bb - (double)bh[i]);
        } else {
            bh[i] = (float)((double)b - (n.mean[i % S] - (double)n.mh[i % S]) * a);
        }
    }
    __device__ __forceinline__ float z(int i, float x, float d) const {
        if constexpr (SPLIT) return fmaf(x, ah[i], bh[i]) + fmaf(x, al[i], bl[i]);
        else return fmaf(d, ah[i], bh[i]);
    }
};

template <int V, int S, bool SPLIT>
__device__ __forceinline__ Coef<V, SPLIT> coef_of(const Norm<V, S>& n, int chunk, bool on, const float* w, const float* b) {
    Coef<V, SPLIT> c;
#pragma unroll
    for (int i = 0; i < V; ++i) c.set(i, n, on && w ? w[chunk * V + i] : 1.f, on && b ? b[chunk * V + i] : 0.f);
    return c;
}

template <bool EXACT> __device__ __forceinline__ float sigmoid(float z) {
    if constexpr (EXACT) return 1.f / (1.f + expf(-z));
    // 16-bit types: native exp2 and reciprocal, a few 2^-23 off against a result rounded to 2^-9 (bf16) or 2^-12 (fp16)
    else return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}

template <int ACT, bool EXACT> __device__ __forceinline__ float act_fwd(float z) {
    if constexpr (ACT == kRelu) return z < 0.f ? 0.f : z;                    // (keeps a NaN)
    else if constexpr (ACT == kSilu) return z * sigmoid<EXACT>(z);
    else return z;
}

template <int ACT, bool EXACT> __device__ __forceinline__ float act_bwd(float dy, float z) {
    if constexpr (ACT == kRelu) return z > 0.f ? dy : 0.f;
    else if constexpr (ACT == kSilu) { const float s = sigmoid<EXACT>(z); return dy * (s * fmaf(z, 1.f - s, 1.f)); }
    else return dy;
}

// The element passes take the blocks in reverse: the last level of cache still holds what the pass before read last.
template <typename T, int V, int S, int ACT, bool RES>
__global__ __launch_bounds__(256) void gn_apply_kernel(Geo g, const T* __restrict__ x, const T* __restrict__ res,
                                                       const float* __restrict__ w, const float* __restrict__ b,
                                                       const double* __restrict__ stats, T* __restrict__ y) {
    constexpr bool kExact = sizeof(T) == 4;
    const Place p = place(g, (long)gridDim.x - 1 - blockIdx.x);
    if (!p.on) return;
    const Norm<V, S> nc = norm_of<V, S>(g, p, stats);
    const Coef<V, ACT == kRelu> cf = coef_of<V, S, ACT == kRelu>(nc, p.chunk, true, w, b);
    const long col = (long)p.chunk * V, row0 = p.n * g.hw;
    const T *xb = x + row0 * g.ldx + col, *rb = RES ? res + row0 * g.ldr + col : nullptr;
    T* yb = y + row0 * g.C + col;
    Pack<T, V> a[kUnroll], e[kUnroll];
    walk(g, p,
         [&](int u, long r) {
             a[u].load(xb + r * g.ldx);
             if constexpr (RES) e[u].load(rb + r * g.ldr);
         },
         [&](int u, long r) {
             float f[V];
#pragma unroll
             for (int i = 0; i < V; ++i) {
                 const float xv = a[u].get(i);
                 float z = cf.z(i, xv, xv - nc.mh[i % S]);
                 if constexpr (RES) z += e[u].get(i);
                 f[i] = act_fwd<ACT, kExact>(z);
             }
             Pack<T, V>::store(yb + r * g.C, f);
         });
}

// part[n, split, 0 | 1, c] = sum dz | sum dz xhat over the rows of the split
template <typename T, int V, int S, int ACT, bool RES>
__global__ __launch_bounds__(256) void gn_bwd_reduce_kernel(Geo g, const T* __restrict__ dy, const T* __restrict__ x,
                                                            const T* __restrict__ res, const float* __restrict__ w,
                                                            const float* __restrict__ b,
                                                            const double* __restrict__ stats, float* __restrict__ part) {
    constexpr bool kExact = sizeof(T) == 4;
    __shared__ float lds[2 * V * 256];
    const Place p = place(g, blockIdx.x);
    float acc[2 * V];                        // sum dz | sum dz (x - mh): the rest of xhat is put in at the end
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) acc[k] = 0.f;
    Norm<V, S> nc;
    if (p.on) {
        nc = norm_of<V, S>(g, p, stats);
        const Coef<V, ACT == kRelu> cf = coef_of<V, S, ACT == kRelu>(nc, p.chunk, true, w, b);
        const long col = (long)p.chunk * V, row0 = p.n * g.hw;
        const T *xb = x + row0 * g.ldx + col, *db = dy + row0 * g.ldd + col, *rb = RES ? res + row0 * g.ldr + col : nullptr;
        Pack<T, V> a[kUnroll], d[kUnroll], e[kUnroll];
        walk(g, p,
             [&](int u, long r) {
                 a[u].load(xb + r * g.ldx);
                 d[u].load(db + r * g.ldd);
                 if constexpr (RES) e[u].load(rb + r * g.ldr);
             },
             [&](int u, long) {
#pragma unroll
                 for (int i = 0; i < V; ++i) {
                     const float xv = a[u].get(i), xd = xv - nc.mh[i % S];
                     float dz = d[u].get(i);
                     if constexpr (ACT != kNone) {
                         float z = cf.z(i, xv, xd);
                         if constexpr (RES) z += e[u].get(i);
                         dz = act_bwd<ACT, kExact>(dz, z);
                     }
                     acc[i] += dz;
                     acc[V + i] = fmaf(dz, xd, acc[V + i]);
                 }
             });
    }
    join_rows<2 * V, 256>(acc, lds, g.cb, g.rpp, p.lane_row);
    if (p.on && p.lane_row == 0) {
        float* o = part + ((p.n * g.splits + p.split) * 2) * g.C + (long)p.chunk * V;
#pragma unroll
        for (int i = 0; i < V; ++i) { o[i] = acc[i]; o[g.C + i] = fmaf(-nc.ml[i % S], acc[i], acc[V + i]) * nc.rs[i % S]; }
    }
}

// The first mean_blocks blocks: means[n, g] = (m1, m2), a team a group.  The others: dw and db, 16 channels by 64 lines of
// parts a block.
constexpr int kJoin = 1024;

__global__ __launch_bounds__(kJoin) void gn_bwd_join_kernel(Geo g, long groups, int team, int mean_blocks, long lines,
                                                            const float* __restrict__ part, const float* __restrict__ w,
                                                            float* __restrict__ means, float* __restrict__ dw,
                                                            float* __restrict__ db) {
    __shared__ double lds[2][kJoin];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x < mean_blocks) {
        const Team t = team_of<kJoin>(g, groups, team, blockIdx.x);
        const float* base = part + t.n * g.splits * 2 * g.C + t.c0;
        double a = 0.0, q = 0.0;
#pragma unroll 4
        for (int i = t.first; i < t.items; i += t.step) {
            const int s = i / g.cpg, c = i - s * g.cpg;
            const double wc = w ? (double)w[t.c0 + c] : 1.0;
            a += wc * (double)base[(long)s * 2 * g.C + c];
            q += wc * (double)base[(long)s * 2 * g.C + g.C + c];
        }
        a = team_sum(a, team, lds[0]);
        q = team_sum(q, team, lds[1]);
        if (t.on && t.first == 0) {
            const double inv = 1.0 / ((double)g.hw * g.cpg);
            means[2 * t.gi] = (float)(a * inv);
            means[2 * t.gi + 1] = (float)(q * inv);
        }
        return;
    }
    const int c = ((int)blockIdx.x - mean_blocks) * 16 + (tid & 15);
    double s1 = 0.0, s2 = 0.0;
    if (c < g.C)
#pragma unroll 8
        for (long k = tid >> 4; k < lines; k += kJoin / 16) {
            s1 += (double)part[2 * k * g.C + c];
            s2 += (double)part[(2 * k + 1) * g.C + c];
        }
    lds[0][tid] = s1;
    lds[1][tid] = s2;
    for (int s = kJoin / 2; s >= 16; s >>= 1) {
        __syncthreads();
        if (tid < s) { lds[0][tid] += lds[0][tid + s]; lds[1][tid] += lds[1][tid + s]; }
    }
    if (tid < 16 && c < g.C) {
        if (dw) dw[c] = (float)lds[1][tid];
        if (db) db[c] = (float)lds[0][tid];
    }
}

template <typename T, int V, int S, int ACT, bool RES>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(Geo g, const T* __restrict__ dy, const T* __restrict__ x,
                                                           const T* __restrict__ res, const float* __restrict__ w,
                                                           const float* __restrict__ b, const double* __restrict__ stats,
                                                           const float* __restrict__ means, T* __restrict__ dx,
                                                           T* __restrict__ dres) {
    constexpr bool kExact = sizeof(T) == 4;
    const Place p = place(g, (long)gridDim.x - 1 - blockIdx.x);
    if (!p.on) return;
    const Norm<V, S> nc = norm_of<V, S>(g, p, stats);
    const Coef<V, ACT == kRelu> cf = coef_of<V, S, ACT == kRelu>(nc, p.chunk, true, w, b);
    float wc[V], m1[S], k2[S];               // dx = rs ((w dz - m1) - (x - mh) k2)
#pragma unroll
    for (int i = 0; i < V; ++i) wc[i] = w ? w[p.chunk * V + i] : 1.f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const float* m = means + 2 * (p.n * g.G + (p.chunk * V + i) / g.cpg);
        k2[i] = nc.rs[i] * m[1];
        m1[i] = fmaf(-nc.ml[i], k2[i], m[0]);
    }
    const long col = (long)p.chunk * V, row0 = p.n * g.hw;
    const T *xb = x + row0 * g.ldx + col, *db = dy + row0 * g.ldd + col, *rb = RES ? res + row0 * g.ldr + col : nullptr;
    T *ob = dx + row0 * g.C + col, *hb = RES ? dres + row0 * g.C + col : nullptr;
    Pack<T, V> a[kUnroll], d[kUnroll], e[kUnroll];
    walk(g, p,
         [&](int u, long r) {
             a[u].load(xb + r * g.ldx);
             d[u].load(db + r * g.ldd);
             if constexpr (RES) e[u].load(rb + r * g.ldr);
         },
         [&](int u, long r) {
             float f[V], h[V];
#pragma unroll
             for (int i = 0; i < V; ++i) {
                 const float xv = a[u].get(i), xd = xv - nc.mh[i % S];
                 float dz = d[u].get(i);
                 if constexpr (ACT != kNone) {
                     float z = cf.z(i, xv, xd);
                     if constexpr (RES) z += e[u].get(i);
                     dz = act_bwd<ACT, kExact>(dz, z);
                 }
                 h[i] = dz;
                 f[i] = nc.rs[i % S] * fmaf(-xd, k2[i % S], wc[i] * dz - m1[i % S]);
             }
             Pack<T, V>::store(ob + r * g.C, f);
             if constexpr (RES) Pack<T, V>::store(hb + r * g.C, h);
         });
}

// ------------------------------------------------------------------------------------------------ groups that fit a block
// Where a group's map fits the registers of one block (at most held<V>(RES) packs or elements for each of its 512 threads),
// the block reads it once, takes the statistics from its registers (the mean first, then the squared differences from it) and
// writes the result: one launch forward, two backward, and no second read.  A group's rows are pieces of cpg elements, often
// less than a cache line: the groups that share lines run next to each other on one XCD, whose L2 then reads each line once
// (counted: 67 MB of a 67 MB map).  512 channels of 16 x 64 x 64 in 32 groups, bf16, ReLU, against the passes above: forward
// 38 us (51; 76 without that order) with inputs in the last level of cache and 50 (62) without, backward 72 (78) and 84..88
// (79).  Where inputs lie is not known here, and both directions together are faster in one block either way.
// A CU holds one block, so loads, sums and stores of a block follow one another; two blocks (128 registers) took 58 us
// forward without cached inputs, 1,024 threads spilled.
constexpr int kBlock = 512;
// Packs (a residual is one more operand) or single elements that a thread holds.  Single ones serve groups that split packs
// and rows off 16 bytes, up to 8,192 elements a group, in pieces of a few bytes, which one block reads in less time than
// three launches take: 3 x 48 channels of 2,720 positions, fp32, 16 groups, forward and backward 24 us (34 in passes); 32
// images of them 52 (54); 16 elements a thread, since 40 (20,480 a group) took 70 us where the passes take 49.
template <int V> constexpr int held(bool res) { return V == 1 ? 16 : res ? 8 : 16; }

__device__ __forceinline__ unsigned xcd_order(unsigned id, unsigned total) {
    const unsigned x = id & 7, i = id >> 3, q = total >> 3, r = total & 7;
    return x * q + (x < r ? x : r) + i;
}

struct Slab { long n; int chunk, row, rows; bool on; };

__device__ __forceinline__ Slab slab_of(const Geo& g, long id) {
    const int cw = g.cv;                                  // packs of a group's row (make_slab)
    Slab s;
    s.n = id / g.G;
    s.rows = kBlock / cw;
    s.row = (int)threadIdx.x / cw;
    s.chunk = (int)(id % g.G) * cw + (int)threadIdx.x % cw;
    s.on = s.row < s.rows;
    return s;
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < kBlock / 64; ++i) t += lds[i];
    return t;
}

template <typename T, int V, int K>
__device__ __forceinline__ void slab_load(Pack<T, V> (&a)[K], const T* base, long ld, const Geo& g, const Slab& s) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long r = s.row + (long)k * s.rows;
        if (s.on && r < g.hw) a[k].load(base + (s.n * g.hw + r) * ld + (long)s.chunk * V);
    }
}

template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(kBlock) void gn_slab_fwd_kernel(Geo g, const T* __restrict__ x, const T* __restrict__ res,
                                                             const float* __restrict__ w, const float* __restrict__ b,
                                                             T* __restrict__ y, double* __restrict__ stats) {
    constexpr bool kExact = sizeof(T) == 4;
    constexpr int K = held<V>(RES);
    __shared__ double lds[kBlock / 64];
    const long id = xcd_order(blockIdx.x, gridDim.x);
    const Slab s = slab_of(g, id);
    Pack<T, V> a[K], e[K];
    slab_load<T, V, K>(a, x, g.ldx, g, s);
    if constexpr (RES) slab_load<T, V, K>(e, res, g.ldr, g, s);
    const double inv = 1.0 / ((double)g.hw * g.cpg);
    // differences from the thread's own first element, so that a mean far above the spread costs no bits
    const float first = s.on && s.row < g.hw ? a[0].get(0) : 0.f;
    float sum = 0.f;
    int held = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (s.on && s.row + (long)k * s.rows < g.hw) {
            held += V;
#pragma unroll
            for (int i = 0; i < V; ++i) sum += a[k].get(i) - first;
        }
    const double mean = block_sum((double)sum + (double)held * (double)first, lds) * inv;
    Norm<V, 1> nc;
    nc.mean[0] = mean;
    nc.mh[0] = (float)mean;
    nc.ml[0] = (float)(mean - (double)nc.mh[0]);
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (s.on && s.row + (long)k * s.rows < g.hw)
#pragma unroll
            for (int i = 0; i < V; ++i) { const float d = (a[k].get(i) - nc.mh[0]) - nc.ml[0]; sq = fmaf(d, d, sq); }
    const double rstd = inv_std(g, block_sum((double)sq, lds) * inv);
    if (threadIdx.x == 0) { stats[2 * id] = mean; stats[2 * id + 1] = rstd; }
    if (!s.on) return;
    nc.rstd[0] = rstd;
    const Coef<V, ACT == kRelu> cf = coef_of<V, 1, ACT == kRelu>(nc, s.chunk, true, w, b);
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long r = s.row + (long)k * s.rows;
        if (r < g.hw) {
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xv = a[k].get(i);
                float z = cf.z(i, xv, xv - nc.mh[0]);
                if constexpr (RES) z += e[k].get(i);
                f[i] = act_fwd<ACT, kExact>(z);
            }
            Pack<T, V>::store(y + (s.n * g.hw + r) * g.C + (long)s.chunk * V, f);
        }
    }
}

// part[n, 0 | 1, c] = sum dz | sum dz xhat of the image, for dw and db
template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(kBlock) void gn_slab_bwd_kernel(Geo g, const T* __restrict__ dy, const T* __restrict__ x,
                                                             const T* __restrict__ res, const float* __restrict__ w,
                                                             const float* __restrict__ b,
                                                             const double* __restrict__ stats, T* __restrict__ dx,
                                                             T* __restrict__ dres, float* __restrict__ part) {
    constexpr bool kExact = sizeof(T) == 4, kAct = ACT != kNone;
    constexpr int K = held<V>(RES);
    __shared__ float lds[2 * V * kBlock];
    __shared__ double sums[kBlock / 64];
    const long id = xcd_order(blockIdx.x, gridDim.x);
    const Slab s = slab_of(g, id);
    Pack<T, V> a[K], d[K], e[K];
    slab_load<T, V, K>(a, x, g.ldx, g, s);
    slab_load<T, V, K>(d, dy, g.ldd, g, s);
    if constexpr (RES) slab_load<T, V, K>(e, res, g.ldr, g, s);
    Norm<V, 1> nc;
    nc.mean[0] = stats[2 * id];
    nc.rstd[0] = stats[2 * id + 1];
    nc.mh[0] = (float)nc.mean[0];
    const float mh = nc.mh[0], ml = (float)(nc.mean[0] - (double)mh), rs = (float)nc.rstd[0];
    const Coef<V, ACT == kRelu> cf = coef_of<V, 1, ACT == kRelu>(nc, s.chunk, s.on, w, b);
    float wc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) wc[i] = s.on && w ? w[s.chunk * V + i] : 1.f;
    auto gradient = [&](int k, int i, float xd) {         // dz
        float dz = d[k].get(i);
        if constexpr (kAct) {
            float z = cf.z(i, a[k].get(i), xd);
            if constexpr (RES) z += e[k].get(i);
            dz = act_bwd<ACT, kExact>(dz, z);
        }
        return dz;
    };
    float acc[2 * V];
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) acc[i] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (s.on && s.row + (long)k * s.rows < g.hw)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xd = a[k].get(i) - mh, dz = gradient(k, i, xd);
                acc[i] += dz;
                acc[V + i] = fmaf(dz, xd, acc[V + i]);
            }
    join_rows<2 * V, kBlock>(acc, lds, g.cv, s.rows, s.row);
    double t1 = 0.0, t2 = 0.0;
    if (s.row == 0) {
        float* o = part + s.n * 2 * g.C + (long)s.chunk * V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            acc[V + i] = fmaf(-ml, acc[i], acc[V + i]) * rs;
            o[i] = acc[i];
            o[g.C + i] = acc[V + i];
            t1 += (double)wc[i] * (double)acc[i];
            t2 += (double)wc[i] * (double)acc[V + i];
        }
    }
    const double inv = 1.0 / ((double)g.hw * g.cpg);
    const float mean1 = (float)(block_sum(t1, sums) * inv), k2 = rs * (float)(block_sum(t2, sums) * inv);
    const float m1 = fmaf(-ml, k2, mean1);
    if (!s.on) return;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const long r = s.row + (long)k * s.rows;
        if (r < g.hw) {
            float f[V], h[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float xd = a[k].get(i) - mh;
                h[i] = gradient(k, i, xd);
                f[i] = rs * fmaf(-xd, k2, wc[i] * h[i] - m1);
            }
            const long at = (s.n * g.hw + r) * g.C + (long)s.chunk * V;
            Pack<T, V>::store(dx + at, f);
            if constexpr (RES) Pack<T, V>::store(dres + at, h);
        }
    }
}

// At most two blocks for each of the 256 CUs, one after the other: a block takes 4 us forward and 10 backward however little
// it holds.  64 x 512 x 7 x 7, bf16, ReLU, forward and backward: 64 groups 235 us against 41 in passes, 32 groups 118 against
// 39; 16 images, 64 groups 65 against 39.
template <int V> bool fits_slab(const Geo& g, long groups, bool res) {
    return groups <= 512 && g.cpg % V == 0 && g.cpg / V <= kBlock && g.hw <= (long)held<V>(res) * (kBlock / (g.cpg / V));
}

Geo make_slab(Geo g, int V) {
    g.cv = g.cpg / V;
    g.splits = 1;
    return g;
}

Geo make_geo(long images, long hw, int C, int G, int V, float eps, long ldx, long ldr, long ldd) {
    Geo g;
    g.hw = hw; g.C = C; g.G = G; g.cpg = C / G; g.eps = eps;
    g.cv = C / V;
    g.cblocks = (g.cv + 255) / 256;
    g.cb = (g.cv + g.cblocks - 1) / g.cblocks;
    g.rpp = 256 / g.cb;
    // about 1024 blocks in all (four to a CU), and no range shorter than two unrolled steps of the block's rows
    const long per = (long)images * g.cblocks;
    long splits = (1024 + per - 1) / per;
    const long most = (hw + (long)g.rpp * kUnroll * 2 - 1) / ((long)g.rpp * kUnroll * 2);
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    g.rows = (hw + splits - 1) / splits;
    g.splits = (int)((hw + g.rows - 1) / g.rows);
    g.ldx = ldx; g.ldr = ldr; g.ldd = ldd;
    return g;
}

// threads of a team, by the group's items: 16,384 groups of two items take 7 us with 16 threads each, 17 with 64
int team_of_group(const Geo& g) { const long items = (long)g.cpg * g.splits; return items > 64 ? 256 : items > 16 ? 64 : 16; }

long team_blocks(long groups, int team, int threads) { return (groups * team + threads - 1) / threads; }

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// elements of a pack: 16 bytes where every row of every operand starts on 16 bytes, single elements otherwise
int pack_width(int esize, int C, long ldx, long ldr, long ldd, const void* a, const void* b, const void* c, const void* d,
               const void* e) {
    const int V = 16 / esize;
    const bool ok = C % V == 0 && ldx % V == 0 && ldr % V == 0 && ldd % V == 0 && aligned16(a) && aligned16(b) &&
                    aligned16(c) && aligned16(d) && aligned16(e);
    return ok ? V : 1;
}

bool bad_shape(long images, long hw, int C, int G, long ldx, long ldr, long ldd) {
    return images <= 0 || hw <= 0 || C <= 0 || G <= 0 || C % G != 0 || ldx < C || ldr < C || ldd < C;
}

struct Fwd {
    const void *x, *res; const float *w, *b; void* y; double* stats; float* ws;
    hipStream_t stream;
};

template <typename T, int V, int ACT, bool RES> int run_slab_fwd(const Geo& g, long groups, const Fwd& f) {
    gn_slab_fwd_kernel<T, V, ACT, RES><<<dim3((unsigned)groups), kBlock, 0, f.stream>>>(
        make_slab(g, V), (const T*)f.x, (const T*)f.res, f.w, f.b, (T*)f.y, f.stats);
    return DP_LAUNCH_STATUS();
}

template <typename T, int V, int ACT, bool RES>
int run_fwd(const Geo& g, long images, const Fwd& f) {
    const long blocks = images * g.cblocks * g.splits, groups = images * g.G;
    const int team = team_of_group(g);
    if (blocks > 0x7fffffffL || groups > 0x7fffffffL) return -3;
    if (fits_slab<V>(g, groups, RES)) return run_slab_fwd<T, V, ACT, RES>(g, groups, f);
    if (g.cpg % V && fits_slab<1>(g, groups, RES)) return run_slab_fwd<T, 1, ACT, RES>(g, groups, f);
    float* pivot = f.ws;
    float* part = f.ws + images * g.C;
    gn_stats_kernel<T, V><<<dim3((unsigned)blocks), 256, 0, f.stream>>>(g, (const T*)f.x, part, pivot);
    gn_finish_kernel<<<dim3((unsigned)team_blocks(groups, team, 256)), 256, 0, f.stream>>>(g, groups, team, part, pivot, f.stats);
    const auto apply = g.cpg % V == 0 ? gn_apply_kernel<T, V, 1, ACT, RES> : gn_apply_kernel<T, V, V, ACT, RES>;
    apply<<<dim3((unsigned)blocks), 256, 0, f.stream>>>(g, (const T*)f.x, (const T*)f.res, f.w, f.b, f.stats, (T*)f.y);
    return DP_LAUNCH_STATUS();
}

struct Bwd {
    const void *dy, *x, *res; const float *w, *b; const double* stats; void *dx, *dres; float *dw, *db, *ws;
    hipStream_t stream;
};

// blocks for dw and db
unsigned sum_blocks(const Geo& g, const Bwd& f) { return f.dw || f.db ? (unsigned)(((long)g.C + 15) / 16) : 0; }

template <typename T, int V, int ACT, bool RES> int run_slab_bwd(const Geo& g, long images, const Bwd& f) {
    gn_slab_bwd_kernel<T, V, ACT, RES><<<dim3((unsigned)(images * g.G)), kBlock, 0, f.stream>>>(
        make_slab(g, V), (const T*)f.dy, (const T*)f.x, (const T*)f.res, f.w, f.b, f.stats, (T*)f.dx, (T*)f.dres, f.ws);
    const unsigned sums = sum_blocks(g, f);
    if (sums) gn_bwd_join_kernel<<<dim3(sums), kJoin, 0, f.stream>>>(g, 0, 64, 0, images, f.ws, f.w, nullptr, f.dw, f.db);
    return DP_LAUNCH_STATUS();
}

template <typename T, int V, int ACT, bool RES>
int run_bwd(const Geo& g, long images, const Bwd& f) {
    const long blocks = images * g.cblocks * g.splits, groups = images * g.G;
    const int team = team_of_group(g);
    const unsigned sums = sum_blocks(g, f);
    if (blocks > 0x7fffffffL || groups > 0x7fffffffL) return -3;
    if (fits_slab<V>(g, groups, RES)) return run_slab_bwd<T, V, ACT, RES>(g, images, f);
    if (g.cpg % V && fits_slab<1>(g, groups, RES)) return run_slab_bwd<T, 1, ACT, RES>(g, images, f);
    float* means = f.ws;
    float* part = f.ws + 2 * images * g.G;
    const bool one = g.cpg % V == 0;
    const auto reduce = one ? gn_bwd_reduce_kernel<T, V, 1, ACT, RES> : gn_bwd_reduce_kernel<T, V, V, ACT, RES>;
    const auto apply = one ? gn_bwd_apply_kernel<T, V, 1, ACT, RES> : gn_bwd_apply_kernel<T, V, V, ACT, RES>;
    reduce<<<dim3((unsigned)blocks), 256, 0, f.stream>>>(
        g, (const T*)f.dy, (const T*)f.x, (const T*)f.res, f.w, f.b, f.stats, part);
    const unsigned mean_blocks = (unsigned)team_blocks(groups, team, kJoin);
    gn_bwd_join_kernel<<<dim3(mean_blocks + sums), kJoin, 0, f.stream>>>(g, groups, team, (int)mean_blocks, images * g.splits,
                                                                        part, f.w, means, f.dw, f.db);
    apply<<<dim3((unsigned)blocks), 256, 0, f.stream>>>(
        g, (const T*)f.dy, (const T*)f.x, (const T*)f.res, f.w, f.b, f.stats, means, (T*)f.dx, (T*)f.dres);
    return DP_LAUNCH_STATUS();
}

// dtype (0 bf16, 1 fp16, 2 fp32), pack width, activation and residual to template arguments
template <template <typename, int, int, bool> class Run, typename... A>
int dispatch(int dtype, int V, int act, bool res, A&&... a) {
#define DP_GN_ACT(T, W)                                                                                  \
    switch (act * 2 + (int)res) {                                                                        \
        case 0: return Run<T, W, kNone, false>::go(a...);                                                \
        case 1: return Run<T, W, kNone, true>::go(a...);                                                 \
        case 2: return Run<T, W, kRelu, false>::go(a...);                                                \
        case 3: return Run<T, W, kRelu, true>::go(a...);                                                 \
        case 4: return Run<T, W, kSilu, false>::go(a...);                                                \
        case 5: return Run<T, W, kSilu, true>::go(a...);                                                 \
    }                                                                                                    \
    return -1;
    if (dtype == 0) { if (V > 1) { DP_GN_ACT(bf16_raw, 8) } else { DP_GN_ACT(bf16_raw, 1) } }
    if (dtype == 1) { if (V > 1) { DP_GN_ACT(f16, 8) } else { DP_GN_ACT(f16, 1) } }
    if (dtype == 2) { if (V > 1) { DP_GN_ACT(float, 4) } else { DP_GN_ACT(float, 1) } }
#undef DP_GN_ACT
    return -1;
}

template <typename T, int V, int ACT, bool RES> struct RunFwd {
    static int go(const Geo& g, long images, const Fwd& f) { return run_fwd<T, V, ACT, RES>(g, images, f); }
};
template <typename T, int V, int ACT, bool RES> struct RunBwd {
    // without an activation the residual's gradient is dy and nothing needs the residual
    static int go(const Geo& g, long images, const Bwd& f) { return run_bwd<T, V, ACT, RES && ACT != kNone>(g, images, f); }
};

}  // namespace

// Floats of workspace that both directions need (the larger of the two; any alignment gives at most this many).
DP_EXPORT long dp_gn_workspace(long images, long hw, int C, int G, int esize) {
    if (bad_shape(images, hw, C, G, C, C, C) || (esize != 2 && esize != 4)) return -1;
    long most = 0;
    for (int V : {16 / esize, 1}) {
        if (C % V) continue;
        const Geo g = make_geo(images, hw, C, G, V, 0.f, C, C, C);
        const long need = images * g.splits * 2 * C + (images * (long)C > 2 * images * G ? images * (long)C : 2 * images * G);
        most = need > most ? need : most;
    }
    return most;
}

DP_EXPORT int dp_gn_fwd(const void* x, const void* res, const float* w, const float* b, void* y, double* stats, float* ws,
                        long images, long hw, int C, int G, long ldx, long ldr, float eps, int act, int dtype, void* stream) {
    if (bad_shape(images, hw, C, G, ldx, ldr, C) || !x || !y || !stats || !ws || act < 0 || act > 2 || dtype < 0 || dtype > 2)
        return -2;
    const int V = pack_width(dtype == 2 ? 4 : 2, C, ldx, ldr, C, x, res, y, nullptr, nullptr);
    const Geo g = make_geo(images, hw, C, G, V, eps, ldx, ldr, C);
    return dispatch<RunFwd>(dtype, V, act, res != nullptr, g, images, Fwd{x, res, w, b, y, stats, ws, (hipStream_t)stream});
}

// res: the forward's residual (needed where an activation follows it; its gradient then goes to dres)
DP_EXPORT int dp_gn_bwd(const void* dy, const void* x, const void* res, const float* w, const float* b, const double* stats,
                        void* dx, void* dres, float* dw, float* db, float* ws, long images, long hw, int C, int G, long ldx,
                        long ldr, long ldd, int act, int dtype, void* stream) {
    if (bad_shape(images, hw, C, G, ldx, ldr, ldd) || !dy || !x || !dx || !stats || !ws || act < 0 || act > 2 || dtype < 0 ||
        dtype > 2 || (res && act != kNone && !dres))
        return -2;
    const int V = pack_width(dtype == 2 ? 4 : 2, C, ldx, ldr, ldd, dy, x, res, dx, dres);
    const Geo g = make_geo(images, hw, C, G, V, 0.f, ldx, ldr, ldd);
    return dispatch<RunBwd>(dtype, V, act, res != nullptr, g, images,
                            Bwd{dy, x, res, w, b, stats, dx, dres, dw, db, ws, (hipStream_t)stream});
}
