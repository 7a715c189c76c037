// Dropout whose mask is a function of (seed, position): forward and backward both compute it, nothing is stored.
//
//   y = keep(i) x s (+ residual),   dx = keep(i) dy s,   s = 1 / (1 - thr / 65536),  thr = p in steps of 1 / 65536
//
// keep(i): Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011).
// Block j of eight elements has the counter (j, j >> 32, 0, 0) and the 64-bit seed as its key; each of the four words
// decides two elements, the low half the first: kept where the half is at least thr.
//
// Bound by memory: one read and one write an element (two reads with a residual); ten rounds are 20 wide integer products
// for eight elements.  16 x 256 x 129 x 129, bf16: 78 us with a residual (three maps, 409 MB: 5.2 TB/s), 45 us without
// (6.1 TB/s); a copy of 2 GiB moves 4.9 TB/s: the generator is hidden.
#include "common.h"

namespace {

typedef _Float16 f16;

struct Key {
    unsigned lo, hi;
    const long long* seed;     // device seed (then lo / hi are not used), or null
    const unsigned* word;      // device word mixed into the key (captured training steps: common.h), or null
};

__device__ __forceinline__ uint4 philox10(unsigned long long block, unsigned k0, unsigned k1) {
    unsigned a = (unsigned)block, b = (unsigned)(block >> 32), c = 0, d = 0;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long l = (unsigned long long)a * 0xD2511F53u, h = (unsigned long long)c * 0xCD9E8D57u;
        a = (unsigned)(h >> 32) ^ b ^ k0;
        b = (unsigned)h;
        c = (unsigned)(l >> 32) ^ d ^ k1;
        d = (unsigned)l;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(a, b, c, d);
}

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<bf16_raw>(bf16_raw v) { return bf2f(v); }
template <> __device__ __forceinline__ float to_f<f16>(f16 v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_raw from_f<bf16_raw>(float v) { return f2bf(v); }
template <> __device__ __forceinline__ f16 from_f<f16>(float v) { return (f16)v; }

template <typename T> struct Eight { T v[8]; };

// eight elements from p, as 16-byte accesses where p allows them; beyond count they are neither read nor written
template <typename T, bool ALIGNED> __device__ __forceinline__ Eight<T> load8(const T* p, long left) {
    Eight<T> r;
    if (ALIGNED && left >= 8) {
        uint4 u[sizeof(T) / 2];
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) u[k] = reinterpret_cast<const uint4*>(p)[k];
        __builtin_memcpy(&r, u, sizeof(r));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = i < left ? p[i] : T(0);
    }
    return r;
}

template <typename T, bool ALIGNED, bool RES>
__global__ __launch_bounds__(256) void dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
                                                      long count, unsigned thr, float scale, Key key) {
    unsigned k0 = key.lo, k1 = key.hi;
    if (key.seed) { const unsigned long long s = (unsigned long long)key.seed[0]; k0 = (unsigned)s; k1 = (unsigned)(s >> 32); }
    if (key.word) k1 ^= key.word[0] * 0x9E3779B9u;
    const long blocks = (count + 7) / 8;
    for (long j = (long)blockIdx.x * 256 + threadIdx.x; j < blocks; j += (long)gridDim.x * 256) {
        const long left = count - j * 8;
        const Eight<T> a = load8<T, ALIGNED>(x + j * 8, left);
        Eight<T> e;
        if constexpr (RES) e = load8<T, ALIGNED>(res + j * 8, left);
        const uint4 r = philox10((unsigned long long)j, k0, k1);
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
        Eight<T> o;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const unsigned half = (i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
            float f = half >= thr ? to_f(a.v[i]) * scale : 0.f;
            if constexpr (RES) f += to_f(e.v[i]);
            o.v[i] = from_f<T>(f);
        }
        if (ALIGNED && left >= 8) {
            uint4 u[sizeof(T) / 2];
            __builtin_memcpy(u, &o, sizeof(o));
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(y + j * 8)[k] = u[k];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) y[j * 8 + i] = o.v[i];
        }
    }
}

template <typename T>
int launch(const void* x, const void* res, void* y, long count, unsigned thr, float scale, const Key& key, hipStream_t st) {
    const bool al = (((uintptr_t)x | (uintptr_t)res | (uintptr_t)y) & 15) == 0;
    const long need = (count + 2047) / 2048;
    const dim3 grid((unsigned)(need < 8192 ? need : 8192));
    const T *xt = (const T*)x, *rt = (const T*)res;
    T* yt = (T*)y;
    if (al && res) dropout_kernel<T, true, true><<<grid, 256, 0, st>>>(xt, rt, yt, count, thr, scale, key);
    else if (al) dropout_kernel<T, true, false><<<grid, 256, 0, st>>>(xt, rt, yt, count, thr, scale, key);
    else if (res) dropout_kernel<T, false, true><<<grid, 256, 0, st>>>(xt, rt, yt, count, thr, scale, key);
    else dropout_kernel<T, false, false><<<grid, 256, 0, st>>>(xt, rt, yt, count, thr, scale, key);
    return DP_LAUNCH_STATUS();
}

}  // namespace

// use_word: mix the captured step's device word into the key (seeds that the framework draws; a caller's own seed is
// taken as it is)
DP_EXPORT int dp_dropout(const void* x, const void* res, void* y, long count, unsigned thr, unsigned long long seed,
                         const long long* seed_dev, int use_word, int dtype, void* stream) {
    if (!x || !y || count <= 0 || thr > 65536 || dtype < 0 || dtype > 2) return -2;
    const float scale = thr < 65536 ? 65536.f / (65536.f - (float)thr) : 0.f;
    const Key key{(unsigned)seed, (unsigned)(seed >> 32), seed_dev, use_word ? g_dp_drop_word : nullptr};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == 0) return launch<bf16_raw>(x, res, y, count, thr, scale, key, st);
    if (dtype == 1) return launch<f16>(x, res, y, count, thr, scale, key, st);
    return launch<float>(x, res, y, count, thr, scale, key, st);
}
