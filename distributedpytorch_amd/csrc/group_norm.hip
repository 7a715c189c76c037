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
// Precision.  Statistics are sums of differences from a per-channel pivot (the mean of four spread positions), so a map
// whose mean is far larger than its spread loses nothing to cancellation; channels are joined by their means and their
// squared deviations (all terms positive) in 64 bits.  z is formed as x a + b with a and b split into a rounded value
// and its remainder: its error is relative to z itself, so an activation's border falls where the definition puts it.
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
template <typename T, int V> struct Pack { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    Pack<T, V> r;
    if constexpr (V == 1) r.v[0] = *p;
    else { static_assert(sizeof(T) * V == 16, "one 16-byte access"); r = __builtin_bit_cast(Pack<T, V>, *reinterpret_cast<const uint4*>(p)); }
    return r;
}
template <typename T, int V> __device__ __forceinline__ void store_pack(T* p, const float* f) {
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = from_f<T>(f[i]);
    if constexpr (V == 1) *p = r.v[0];
    else *reinterpret_cast<uint4*>(p) = __builtin_bit_cast(uint4, r);
}

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

__device__ __forceinline__ Place place(const Geo& g) {
    Place p;
    const long id = blockIdx.x;
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

// sum of acc[0..K) over the rpp threads that share a pack; the result is left with the threads of lane_row 0
template <int K> __device__ __forceinline__ void join_rows(float* acc, float* lds, const Geo& g, const Place& p) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int k = 0; k < K; ++k) lds[k * 256 + tid] = acc[k];
    int s = 1;
    while (s < g.rpp) s <<= 1;
    for (s >>= 1; s > 0; s >>= 1) {
        __syncthreads();
        if (p.lane_row < s && p.lane_row + s < g.rpp)
#pragma unroll
            for (int k = 0; k < K; ++k) lds[k * 256 + tid] += lds[k * 256 + tid + s * g.cb];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) acc[k] = lds[k * 256 + tid];
}

constexpr int kUnroll = 4;   // packs in flight per thread and operand

template <typename T, int V>
__global__ __launch_bounds__(256) void gn_stats_kernel(Geo g, const T* __restrict__ x, float* __restrict__ part,
                                                       float* __restrict__ pivot) {
    __shared__ float lds[2 * V * 256];
    const Place p = place(g);
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
            const Pack<T, V> a = load_pack<T, V>(base + (g.hw * s / 4) * g.ldx);
#pragma unroll
            for (int i = 0; i < V; ++i) pv[i] += 0.25f * to_f(a.v[i]);
        }
        if (p.split == 0 && p.lane_row == 0)
#pragma unroll
            for (int i = 0; i < V; ++i) pivot[p.n * g.C + (long)p.chunk * V + i] = pv[i];
        for (long r = p.row; r < p.row_end; r += (long)kUnroll * g.rpp) {
            Pack<T, V> a[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (r + u * g.rpp < p.row_end) a[u] = load_pack<T, V>(base + (r + u * g.rpp) * g.ldx);
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (r + u * g.rpp < p.row_end)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float d = to_f(a[u].v[i]) - pv[i];
                        acc[i] += d;
                        acc[V + i] = fmaf(d, d, acc[V + i]);
                    }
        }
    }
    join_rows<2 * V>(acc, lds, g, p);
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

// one wave per (image, group): stats[n, g] = (mean, rstd)
__global__ __launch_bounds__(256) void gn_finish_kernel(Geo g, long waves, const float* __restrict__ part,
                                                        const float* __restrict__ pivot, double* __restrict__ stats) {
    const long w = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (w >= waves) return;
    const long n = w / g.G;
    const int c0 = (int)(w % g.G) * g.cpg;
    const double inv = 1.0 / (double)g.hw;
    double sm = 0.0;
    for (int c = lane; c < g.cpg; c += 64) {
        const float* q = part + n * g.splits * 2 * g.C + c0 + c;
        double s1 = 0.0;
        for (int s = 0; s < g.splits; ++s) s1 += (double)q[(long)s * 2 * g.C];
        sm += (double)pivot[n * g.C + c0 + c] + s1 * inv;
    }
    const double mean = wave_sum_d(sm) / g.cpg;
    double m2 = 0.0;
    for (int c = lane; c < g.cpg; c += 64) {
        const float* q = part + n * g.splits * 2 * g.C + c0 + c;
        double s1 = 0.0, s2 = 0.0;
        for (int s = 0; s < g.splits; ++s) { s1 += (double)q[(long)s * 2 * g.C]; s2 += (double)q[(long)s * 2 * g.C + g.C]; }
        const double d = (double)pivot[n * g.C + c0 + c] + s1 * inv - mean;
        const double own = s2 - s1 * s1 * inv;
        m2 += (own > 0.0 ? own : (own != own ? own : 0.0)) + d * d * (double)g.hw;      // (a NaN stays one)
    }
    m2 = wave_sum_d(m2);
    if (lane == 0) {
        const double var = m2 / ((double)g.hw * g.cpg);
        stats[2 * w] = mean;
        stats[2 * w + 1] = 1.0 / sqrt(var + (double)g.eps);
    }
}

// per-channel constants of one thread
template <int V> struct Coef { float ah[V], al[V], bh[V], bl[V]; };        // z = x a + b (+ residual)

template <int V>
__device__ __forceinline__ Coef<V> coef(const Geo& g, const Place& p, const double* stats, const float* w, const float* b) {
    Coef<V> c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int ch = p.chunk * V + i;
        const double* st = stats + 2 * (p.n * g.G + ch / g.cpg);
        const double a = (w ? (double)w[ch] : 1.0) * st[1], bb = (b ? (double)b[ch] : 0.0) - st[0] * a;
        c.ah[i] = (float)a; c.al[i] = (float)(a - (double)c.ah[i]);
        c.bh[i] = (float)bb; c.bl[i] = (float)(bb - (double)c.bh[i]);
    }
    return c;
}

// Near z = 0 the first product leaves z almost exactly and the second adds what the rounded coefficients left out.
__device__ __forceinline__ float affine(float x, float ah, float al, float bh, float bl) {
    return fmaf(x, ah, bh) + fmaf(x, al, bl);
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

template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(256) void gn_apply_kernel(Geo g, const T* __restrict__ x, const T* __restrict__ res,
                                                       const float* __restrict__ w, const float* __restrict__ b,
                                                       const double* __restrict__ stats, T* __restrict__ y) {
    constexpr bool kExact = sizeof(T) == 4;
    const Place p = place(g);
    if (!p.on) return;
    const Coef<V> cf = coef<V>(g, p, stats, w, b);
    const long col = (long)p.chunk * V, row0 = p.n * g.hw;
    for (long r = p.row; r < p.row_end; r += (long)kUnroll * g.rpp) {
        Pack<T, V> a[kUnroll], e[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long q = r + u * g.rpp;
            if (q < p.row_end) {
                a[u] = load_pack<T, V>(x + (row0 + q) * g.ldx + col);
                if constexpr (RES) e[u] = load_pack<T, V>(res + (row0 + q) * g.ldr + col);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long q = r + u * g.rpp;
            if (q < p.row_end) {
                float f[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float z = affine(to_f(a[u].v[i]), cf.ah[i], cf.al[i], cf.bh[i], cf.bl[i]);
                    if constexpr (RES) z += to_f(e[u].v[i]);
                    f[i] = act_fwd<ACT, kExact>(z);
                }
                store_pack<T, V>(y + (row0 + q) * g.C + col, f);
            }
        }
    }
}

template <int V> struct Norm { float mh[V], ml[V], rs[V]; };               // xhat = (x - mean) rstd

template <int V> __device__ __forceinline__ Norm<V> norm_coef(const Geo& g, const Place& p, const double* stats) {
    Norm<V> c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const double* st = stats + 2 * (p.n * g.G + (p.chunk * V + i) / g.cpg);
        c.mh[i] = (float)st[0]; c.ml[i] = (float)(st[0] - (double)c.mh[i]); c.rs[i] = (float)st[1];
    }
    return c;
}

__device__ __forceinline__ float xhat_of(float x, float mh, float ml, float rs) { return ((x - mh) - ml) * rs; }

// part[n, split, 0 | 1, c] = sum dz | sum dz xhat over the rows of the split
template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(256) void gn_bwd_reduce_kernel(Geo g, const T* __restrict__ dy, const T* __restrict__ x,
                                                            const T* __restrict__ res, const float* __restrict__ w,
                                                            const float* __restrict__ b,
                                                            const double* __restrict__ stats, float* __restrict__ part) {
    constexpr bool kExact = sizeof(T) == 4;
    __shared__ float lds[2 * V * 256];
    const Place p = place(g);
    float acc[2 * V];
#pragma unroll
    for (int k = 0; k < 2 * V; ++k) acc[k] = 0.f;
    if (p.on) {
        const Coef<V> cf = coef<V>(g, p, stats, w, b);
        const Norm<V> nc = norm_coef<V>(g, p, stats);
        const long col = (long)p.chunk * V, row0 = p.n * g.hw;
        for (long r = p.row; r < p.row_end; r += (long)kUnroll * g.rpp) {
            Pack<T, V> a[kUnroll], d[kUnroll], e[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const long q = r + u * g.rpp;
                if (q < p.row_end) {
                    a[u] = load_pack<T, V>(x + (row0 + q) * g.ldx + col);
                    d[u] = load_pack<T, V>(dy + (row0 + q) * g.ldd + col);
                    if constexpr (RES && ACT != kNone) e[u] = load_pack<T, V>(res + (row0 + q) * g.ldr + col);
                }
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (r + u * g.rpp < p.row_end)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float xv = to_f(a[u].v[i]);
                        float dz = to_f(d[u].v[i]);
                        if constexpr (ACT != kNone) {
                            float z = affine(xv, cf.ah[i], cf.al[i], cf.bh[i], cf.bl[i]);
                            if constexpr (RES) z += to_f(e[u].v[i]);
                            dz = act_bwd<ACT, kExact>(dz, z);
                        }
                        acc[i] += dz;
                        acc[V + i] = fmaf(dz, xhat_of(xv, nc.mh[i], nc.ml[i], nc.rs[i]), acc[V + i]);
                    }
        }
    }
    join_rows<2 * V>(acc, lds, g, p);
    if (p.on && p.lane_row == 0) {
        float* o = part + ((p.n * g.splits + p.split) * 2) * g.C + (long)p.chunk * V;
#pragma unroll
        for (int i = 0; i < V; ++i) { o[i] = acc[i]; o[g.C + i] = acc[V + i]; }
    }
}

// blocks [0, gblocks): one wave per (image, group) -> means[n, g] = (m1, m2); the rest: one thread per channel -> dw, db
__global__ __launch_bounds__(256) void gn_bwd_finish_kernel(Geo g, long images, int gblocks, const float* __restrict__ part,
                                                            const float* __restrict__ w, float* __restrict__ means,
                                                            float* __restrict__ dw, float* __restrict__ db) {
    if ((int)blockIdx.x < gblocks) {
        const long wv = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
        const int lane = threadIdx.x & 63;
        if (wv >= images * g.G) return;
        const long n = wv / g.G;
        const int c0 = (int)(wv % g.G) * g.cpg;
        double a = 0.0, q = 0.0;
        for (int c = lane; c < g.cpg; c += 64) {
            const float* s = part + n * g.splits * 2 * g.C + c0 + c;
            double s1 = 0.0, s2 = 0.0;
            for (int k = 0; k < g.splits; ++k) { s1 += (double)s[(long)k * 2 * g.C]; s2 += (double)s[(long)k * 2 * g.C + g.C]; }
            const double wc = w ? (double)w[c0 + c] : 1.0;
            a += wc * s1; q += wc * s2;
        }
        a = wave_sum_d(a); q = wave_sum_d(q);
        if (lane == 0) {
            const double inv = 1.0 / ((double)g.hw * g.cpg);
            means[2 * wv] = (float)(a * inv);
            means[2 * wv + 1] = (float)(q * inv);
        }
        return;
    }
    const int c = ((int)blockIdx.x - gblocks) * 256 + threadIdx.x;
    if (c >= g.C) return;
    double s1 = 0.0, s2 = 0.0;
    for (long k = 0; k < images * g.splits; ++k) { s1 += (double)part[2 * k * g.C + c]; s2 += (double)part[(2 * k + 1) * g.C + c]; }
    if (dw) dw[c] = (float)s2;
    if (db) db[c] = (float)s1;
}

template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(Geo g, const T* __restrict__ dy, const T* __restrict__ x,
                                                           const T* __restrict__ res, const float* __restrict__ w,
                                                           const float* __restrict__ b, const double* __restrict__ stats,
                                                           const float* __restrict__ means, T* __restrict__ dx,
                                                           T* __restrict__ dres) {
    constexpr bool kExact = sizeof(T) == 4;
    const Place p = place(g);
    if (!p.on) return;
    const Coef<V> cf = coef<V>(g, p, stats, w, b);
    const Norm<V> nc = norm_coef<V>(g, p, stats);
    float wc[V], m1[V], m2[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int ch = p.chunk * V + i;
        const float* m = means + 2 * (p.n * g.G + ch / g.cpg);
        wc[i] = w ? w[ch] : 1.f; m1[i] = m[0]; m2[i] = m[1];
    }
    const long col = (long)p.chunk * V, row0 = p.n * g.hw;
    for (long r = p.row; r < p.row_end; r += (long)kUnroll * g.rpp) {
        Pack<T, V> a[kUnroll], d[kUnroll], e[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long q = r + u * g.rpp;
            if (q < p.row_end) {
                a[u] = load_pack<T, V>(x + (row0 + q) * g.ldx + col);
                d[u] = load_pack<T, V>(dy + (row0 + q) * g.ldd + col);
                if constexpr (RES && ACT != kNone) e[u] = load_pack<T, V>(res + (row0 + q) * g.ldr + col);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long q = r + u * g.rpp;
            if (q < p.row_end) {
                float f[V], h[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float xv = to_f(a[u].v[i]);
                    float dz = to_f(d[u].v[i]);
                    if constexpr (ACT != kNone) {
                        float z = affine(xv, cf.ah[i], cf.al[i], cf.bh[i], cf.bl[i]);
                        if constexpr (RES) z += to_f(e[u].v[i]);
                        dz = act_bwd<ACT, kExact>(dz, z);
                    }
                    h[i] = dz;
                    // w dz rounded by itself: in a group of one element it then equals m1 and the gradient is zero
                    const float t = __fmul_rn(wc[i], dz) - m1[i];
                    f[i] = nc.rs[i] * fmaf(-xhat_of(xv, nc.mh[i], nc.ml[i], nc.rs[i]), m2[i], t);
                }
                store_pack<T, V>(dx + (row0 + q) * g.C + col, f);
                if constexpr (RES && ACT != kNone) store_pack<T, V>(dres + (row0 + q) * g.C + col, h);
            }
        }
    }
}

Geo make_geo(long images, long hw, int C, int G, int V, float eps, long ldx, long ldr, long ldd) {
    Geo g;
    g.hw = hw; g.C = C; g.G = G; g.cpg = C / G; g.eps = eps;
    g.cv = C / V;
    g.cblocks = (g.cv + 255) / 256;
    g.cb = (g.cv + g.cblocks - 1) / g.cblocks;
    g.rpp = 256 / g.cb;
    // about 2048 blocks in all (eight to a CU), and no range shorter than two unrolled steps of the block's rows
    const long per = (long)images * g.cblocks;
    long splits = (2048 + per - 1) / per;
    const long most = (hw + (long)g.rpp * kUnroll * 2 - 1) / ((long)g.rpp * kUnroll * 2);
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    g.rows = (hw + splits - 1) / splits;
    g.splits = (int)((hw + g.rows - 1) / g.rows);
    g.ldx = ldx; g.ldr = ldr; g.ldd = ldd;
    return g;
}

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

template <typename T, int V, int ACT, bool RES>
int run_fwd(const Geo& g, long images, const Fwd& f) {
    const long blocks = images * g.cblocks * g.splits, waves = images * g.G;
    if (blocks > 0x7fffffffL || (waves + 3) / 4 > 0x7fffffffL) return -3;
    float* pivot = f.ws;
    float* part = f.ws + images * g.C;
    gn_stats_kernel<T, V><<<dim3((unsigned)blocks), 256, 0, f.stream>>>(g, (const T*)f.x, part, pivot);
    gn_finish_kernel<<<dim3((unsigned)((waves + 3) / 4)), 256, 0, f.stream>>>(g, waves, part, pivot, f.stats);
    gn_apply_kernel<T, V, ACT, RES><<<dim3((unsigned)blocks), 256, 0, f.stream>>>(g, (const T*)f.x, (const T*)f.res, f.w, f.b,
                                                                                f.stats, (T*)f.y);
    return DP_LAUNCH_STATUS();
}

struct Bwd {
    const void *dy, *x, *res; const float *w, *b; const double* stats; void *dx, *dres; float *dw, *db, *ws;
    hipStream_t stream;
};

template <typename T, int V, int ACT, bool RES>
int run_bwd(const Geo& g, long images, const Bwd& f) {
    const long blocks = images * g.cblocks * g.splits, gblocks = (images * g.G + 3) / 4;
    if (blocks > 0x7fffffffL || gblocks + g.C > 0x7fffffffL) return -3;
    float* means = f.ws;
    float* part = f.ws + 2 * images * g.G;
    gn_bwd_reduce_kernel<T, V, ACT, RES><<<dim3((unsigned)blocks), 256, 0, f.stream>>>(
        g, (const T*)f.dy, (const T*)f.x, (const T*)f.res, f.w, f.b, f.stats, part);
    gn_bwd_finish_kernel<<<dim3((unsigned)(gblocks + (g.C + 255) / 256)), 256, 0, f.stream>>>(
        g, images, (int)gblocks, part, f.w, means, f.dw, f.db);
    gn_bwd_apply_kernel<T, V, ACT, RES><<<dim3((unsigned)blocks), 256, 0, f.stream>>>(
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
    static int go(const Geo& g, long images, const Bwd& f) { return run_bwd<T, V, ACT, RES>(g, images, f); }
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
