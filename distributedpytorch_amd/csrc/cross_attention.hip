// Attention of one sequence's queries over another's keys and values, forward and backward.
//
//   S = scale q k^T over the keys that take part,  P = softmax(S),  o = P v;   a row without a key gives 0
//   backward, delta = rowsum(do o):   dv = P^T do    dS = P (do v^T - delta) scale    dq = dS k    dk = dS^T q
//
// Heads: q has Hq = Hk * share of them; share neighbouring query heads read one key / value head.  The kernels see, per
// (image, key head), R = Lq * share ROWS (row r: position r / share, head r % share), so shared heads read keys once and
// their gradients add up in the row sum.
//
// Everything runs on v_mfma_f32_32x32x16 with fp32 accumulators and never writes a score to memory: the first product
// leaves rows (or keys) on the lanes and keys (or rows) on the accumulator registers, which, packed in pairs, ARE the
// second operand of the product that contracts over them; the first operand of that product comes out of the row-major
// LDS tile through transposing reads.
//
//   xa_fwd    128 rows a workgroup (32 a wave), keys in blocks of 64 through LDS, running maximum and sum; with few rows
//             the keys are split over workgroups and xa_join puts the parts together
//   xa_dq     128 rows a workgroup, keys in blocks of 64; leaves delta behind for
//   xa_dkv    128 keys a workgroup (32 a wave, their k and v in registers), rows in blocks of 64 through LDS
//   xa_sum    joins the fp32 parts of dq, or of dk and dv, where a long axis was split; one order, no atomics
//
// Measured, all on bf16 and without masks.  A: 16 x 16,641 rows over 1,089 keys, 4 heads of 64 (a training step's decoder).
// B: 4,225 rows over 16,641 keys, 8 heads of 128.  An 8192^3 matrix product of the library reaches 1.24 PFLOP/s.
//   xa_fwd   A 379..409 us (297 GFLOP: 0.73..0.78 PFLOP/s), B 314..328 us (288 GFLOP: 0.88..0.92)
//   xa_dq    A 487..527 us (446 GFLOP: 0.85..0.92)        xa_dkv   A 581..634 us (594 GFLOP: 0.94..1.02)
// What bounds them: in A's forward vector instructions fill 81 % of the issue cycles (a score costs a product-sum, an
// exponential, a sum, half a maximum and half a conversion) and matrix instructions keep the matrix units 45 % busy; dq 64 %
// and 53 %, dkv 48 % and 58 %.  B's forward: 44 % and 50 % with two waves a SIMD, whose latencies show.  LDS is
// busy 22 % (forward) to 43 % (dkv) of the time, without bank conflicts.
//
// P and dS are rounded to the tensors' type before their second product (its operands are 16 bits wide); sums, statistics
// and gradients' accumulators stay in 32 bits.  Masked keys: their scores are replaced, and their k and v rows are staged
// as zeros, so whatever they hold (infinities, NaN) takes no part.
#include "common.h"

namespace {

typedef _Float16 f16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

typedef __attribute__((ext_vector_type(2))) float f32x2v;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

struct Bf {
    typedef bf16_raw raw;
    static __device__ __forceinline__ f32x16 mfma(const uint4& a, const uint4& b, const f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned pair(float lo, float hi) {
        return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2v){lo, hi}, bf16x2));
    }
    static __device__ __forceinline__ void unpair(unsigned u, float& lo, float& hi) {
        lo = __uint_as_float(u << 16); hi = __uint_as_float(u & 0xffff0000u);
    }
};

struct Hf {
    typedef f16 raw;
    static __device__ __forceinline__ f32x16 mfma(const uint4& a, const uint4& b, const f32x16& c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ unsigned pair(float lo, float hi) {
        return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2v){lo, hi}, f16x2));
    }
    static __device__ __forceinline__ void unpair(unsigned u, float& lo, float& hi) {
        lo = (float)__builtin_bit_cast(f16, (unsigned short)u); hi = (float)__builtin_bit_cast(f16, (unsigned short)(u >> 16));
    }
};

// Rows (forward, dq) or keys (dkv) of a workgroup: 4 waves x 32.  Eight waves (half the LDS traffic from L2): dq of A
// 674 us, forward of B 368.
constexpr int kRows = 128;
constexpr int kKeys = 64;        // keys of an LDS block (forward, dq)
constexpr int kStep = 64;        // rows of an LDS block (dkv)
constexpr float kInf = __builtin_huge_valf();

// strides in elements: image, position, head (elements of a head are adjacent)
struct View { long b, l, h; };

struct Att {
    const void *q, *k, *v, *o, *dout;
    void *out, *dq, *dk, *dv;
    float *lse, *delta;              // [B, Hk, R]: log2 of the row's sum of exponentials (+inf: no key), -rowsum(do o)
    const int* lens;                 // [B] keys of each image, or null
    const unsigned char* mask;       // [B, Lk], nonzero = takes part, or null
    long mask_ld;
    View vq, vk, vv, vd;             // of q, k, v and dout (o, dq, dk, dv are dense)
    int B, Lq, Lk, Hk, share, D;
    int R;                           // Lq share
    float scale, c;                  // c = scale log2(e)
    int splits;                      // parts of the split axis
    float* part;                     // their fp32 partial results
};

// A row's log2 of the sum l of its exponentials relative to m: +inf without a key (P = 0 in backward), NaN stays NaN.
__device__ __forceinline__ float log_sum(float m, float l, float c) {
    return l > 0.f ? fmaf(m, c, __builtin_amdgcn_logf(l)) : (l == l ? kInf : l);
}

__device__ __forceinline__ f32x16 splat16(float v) {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = v;
    return z;
}

__device__ __forceinline__ f32x16 zero16() { return splat16(0.f); }

// the larger, or the sum, of the two lanes l and l ^ 32 (a row's two halves), on both of them
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Consecutive workgroups go round the 8 XCDs: give each XCD one contiguous range of the work, so that the workgroups
// that read the same keys share an L2.  Not with lengths: an XCD would get the long images whole, another the empty ones.
__device__ __forceinline__ unsigned xcd_order(unsigned id, unsigned total) {
    const unsigned x = id & 7, i = id >> 3, q = total >> 3, r = total & 7;
    return x * q + (x < r ? x : r) + i;
}

// eight columns of this lane's column pair, rows r0..r0+3 and r1..r1+3 of a row-major tile (two transposing reads)
__device__ __forceinline__ uint4 tr_pair(const unsigned char* a0, const unsigned char* a1) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a0);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a1);
    return __builtin_bit_cast(uint4, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// accumulator registers 8 s .. 8 s + 7 as an operand of 16 contracted entries: lane half h holds entries
// 16 s + 4 h + {0..3} and 16 s + 8 + 4 h + {0..3} of the 32
template <typename E> __device__ __forceinline__ uint4 pack_acc(const f32x16& a, int s) {
    uint4 u;
    u.x = E::pair(a[8 * s + 0], a[8 * s + 1]); u.y = E::pair(a[8 * s + 2], a[8 * s + 3]);
    u.z = E::pair(a[8 * s + 4], a[8 * s + 5]); u.w = E::pair(a[8 * s + 6], a[8 * s + 7]);
    return u;
}

// entry of the 32 that accumulator register r of lane half h belongs to
__device__ __forceinline__ int entry(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// Whether the key of accumulator register i of 32-key tile t takes part, for this lane.  The set is a scalar: its two bits (of
// the lane halves) become a lane mask on the scalar unit, and the select is all that the vector unit does.
__device__ __forceinline__ bool key_on(unsigned long long set, int t, int i) {
    const unsigned bits = (unsigned)(set >> (32 * t));
    const unsigned lo = (unsigned)((int)(bits << (31 - entry(i, 0))) >> 31), hi = (unsigned)((int)(bits << (31 - entry(i, 1))) >> 31);
    return __builtin_amdgcn_inverse_ballot_w64((unsigned long long)hi << 32 | lo);
}

__device__ __forceinline__ float row_max(const f32x16 (&s)[2]) {
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 32; ++i) mx = __builtin_elementwise_maximum(mx, s[i >> 4][i & 15]);
    return mx;
}

// 64-bit sets of the keys that take part, block after block; every wave of the workgroup gets the same.  A block's mask is
// read one block before its set is asked for.
struct KeySets {
    const unsigned char* mask;
    int len;
    bool on;
    __device__ __forceinline__ KeySets(const Att& p, int b, int n) { mask = p.mask ? p.mask + (long)b * p.mask_ld : nullptr; len = n; on = false; }
    __device__ __forceinline__ void ahead(int kb) {
        const int key = kb * 64 + (int)(threadIdx.x & 63);
        if (mask) on = key < len && mask[key] != 0;
    }
    __device__ __forceinline__ unsigned long long of(int kb) const {       // kb: the block of the last ahead()
        if (mask) return __ballot(on);
        const int left = len - kb * 64;
        return left >= 64 ? ~0ull : (1ull << left) - 1;
    }
};

__device__ __forceinline__ int key_count(const Att& p, int b) {
    if (!p.lens) return p.Lk;
    const int n = p.lens[b];
    return n < 0 ? 0 : (n > p.Lk ? p.Lk : n);
}

// Whether a single key of the image's first len takes part: P = 1 whatever its score, so dS and with it dq and dk are zero (but
// a NaN stays one: what the roundings left is multiplied by zero).  Asked by whole waves, and only by those that saw one key.
__device__ __forceinline__ bool single_key(const Att& p, int b, int len) {
    if (!p.mask) return len == 1;
    const unsigned char* mask = p.mask + (long)b * p.mask_ld;
    int n = 0;
    for (int k = 0; k < len && n < 2; k += 512) {
        bool on[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = k + j * 64 + (int)(threadIdx.x & 63);
            on[j] = key < len && mask[key] != 0;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) n += __popcll(__ballot(on[j]));
    }
    return n == 1;
}

// offset of row r of key head hk in a tensor of rows
__device__ __forceinline__ int position(const Att& p, int r) { return p.share == 1 ? r : (int)((unsigned)r / (unsigned)p.share); }

__device__ __forceinline__ long row_at(const Att& p, const View& v, int b, int hk, int r) {
    const int l = position(p, r);
    return b * v.b + l * v.l + (hk * p.share + (r - l * p.share)) * v.h;
}

// the same in a dense [B, Lq, Hq, D] tensor
__device__ __forceinline__ long dense_row(const Att& p, int b, int hk, int r) {
    const int l = position(p, r);
    return (((long)b * p.Lq + l) * (p.Hk * p.share) + hk * p.share + (r - l * p.share)) * p.D;
}

// A tile of 64 rows in LDS.  A row's 16-byte chunks lie permuted (chunk c of row r in slot c ^ swz(r)): rows that share
// banks then keep the same chunk in different ones, for whole-row reads (32 rows, one chunk) and for transposing reads
// (4 rows, 4 chunks) alike.  Piece j of a thread has the place (wave kPieces + j) 1024 + 16 lane, as LDS-DMA writes it: the
// permutation is made by what the lane reads.
template <int DP> struct Tile {
    static constexpr int kPitch = DP == 96 ? 256 : DP * 2;         // bytes of a row: a power of two
    static constexpr int kBytes = 64 * kPitch;
    static constexpr int kPieces = kBytes / 4096;                  // of each of 256 threads
    static __device__ __forceinline__ int swz(int r) {
        return DP == 32 ? (r >> 2) & 3 : DP == 64 ? (r >> 1 & 1) << 2 | (r >> 2 & 3) : (r & 3) << 2 | (r >> 2 & 3);
    }
    static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }
    static __device__ __forceinline__ int place(int j) { return (wave() * kPieces + j) * 1024 + ((int)threadIdx.x & 63) * 16; }
    static __device__ __forceinline__ int row(int j) { return place(j) / kPitch; }
    static __device__ __forceinline__ int col(int j) { return ((place(j) % kPitch / 16) ^ swz(row(j))) * 8; }    // element
};

// Where this lane reads a tile: whole rows (32 of them, 8 elements a lane) and their transposes.
template <int DP> struct Reads {
    int row, tr;
    __device__ __forceinline__ Reads() {
        typedef Tile<DP> L;
        const int lane = threadIdx.x & 63, l31 = lane & 31, h = lane >> 5, q = (lane & 15) >> 2;
        row = l31 * L::kPitch + ((h ^ L::swz(l31)) << 4);
        tr = (4 * h + q) * L::kPitch + (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ L::swz(4 * h + q)) << 4) + (lane & 1) * 8;
    }
    // elements 16 ks + 8 h .. of row 32 t + lane
    __device__ __forceinline__ uint4 rows(const unsigned char* tile, int t, int ks) const {
        return *reinterpret_cast<const uint4*>(tile + t * 32 * Tile<DP>::kPitch + (row ^ (ks << 5)));
    }
    // column 32 t + lane of rows 16 s + 4 h + {0..3} and 16 s + 8 + 4 h + {0..3}
    __device__ __forceinline__ uint4 cols(const unsigned char* tile, int s, int t) const {
        const unsigned char* a = tile + 16 * s * Tile<DP>::kPitch;
        return tr_pair(a + (tr ^ (t << 6)), a + 8 * Tile<DP>::kPitch + (tr ^ (t << 6) ^ 32));
    }
};

constexpr unsigned kOut = 0x80000000u;       // an offset that every buffer descriptor below answers with zeros

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* base, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ void dma(__amdgpu_buffer_rsrc_t from, unsigned char* to, unsigned offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, offset, 0, 0, 0);
}

// Successive tiles of rows, brought a tile ahead of their use.  DMA: straight into LDS; rows and columns that do not exist,
// and masked rows whatever they hold, come as zeros.  Otherwise (strides or head shares that do not fit 32-bit offsets from
// a tile's first row) through registers.
template <typename T, int DP, bool DMA> struct Stream {
    typedef Tile<DP> L;
    unsigned off[DMA ? L::kPieces : 1];
    uint4 u[DMA ? 1 : L::kPieces];
    // byte offset of piece j's row from the tile's first: a multiple of it for keys, position and head for rows
    __device__ __forceinline__ void open(int D, long ld, long head, int share) {
        if constexpr (DMA) {
#pragma unroll
            for (int j = 0; j < L::kPieces; ++j) {
                const int r = L::row(j);
                off[j] = L::col(j) < D ? (unsigned)((r / share * ld + r % share * head + L::col(j)) * 2) : kOut;
            }
        }
    }
    // `set`: the tile's rows that are read
    __device__ __forceinline__ void load(const T* tile, unsigned char* to, unsigned long long set) {
        const __amdgpu_buffer_rsrc_t from = buffer_at(tile, 0x7fffffffu);
        if (set == ~0ull) {
#pragma unroll
            for (int j = 0; j < L::kPieces; ++j) dma(from, to + (L::wave() * L::kPieces + j) * 1024, off[j]);
        } else {
#pragma unroll
            for (int j = 0; j < L::kPieces; ++j)
                dma(from, to + (L::wave() * L::kPieces + j) * 1024, set >> L::row(j) & 1 ? off[j] : kOut);
        }
    }
    __device__ __forceinline__ void put(unsigned char* to) const {
#pragma unroll
        for (int j = 0; j < L::kPieces; ++j) *reinterpret_cast<uint4*>(to + L::place(j)) = u[j];
    }
};

template <typename T, int DP, bool DMA> struct KeyStream : Stream<T, DP, DMA> {
    typedef Tile<DP> L;
    const T* base;
    long ld;
    __device__ __forceinline__ KeyStream(const Att& p, const void* t, const View& v, int b, int hk) {
        base = (const T*)t + b * v.b + hk * v.h;
        ld = v.l;
        this->open(p.D, ld, 0, 1);
    }
    __device__ __forceinline__ void fetch(const Att& p, unsigned char* to, int kb, unsigned long long set) {
        const T* tile = base + (long)kb * kKeys * ld;
        if constexpr (DMA) {
            this->load(tile, to, set);
        } else {
#pragma unroll
            for (int j = 0; j < L::kPieces; ++j) {
                this->u[j] = make_uint4(0, 0, 0, 0);
                if ((set >> L::row(j) & 1) && L::col(j) < p.D)
                    this->u[j] = *reinterpret_cast<const uint4*>(tile + L::row(j) * ld + L::col(j));
            }
        }
    }
};

template <typename T, int DP, bool DMA> struct RowStream : Stream<T, DP, DMA> {
    typedef Tile<DP> L;
    const T* base;
    long step;                               // elements between the first rows of successive tiles (DMA: 64 % share == 0)
    __device__ __forceinline__ RowStream(const Att& p, const void* t, const View& v, int b, int hk) {
        base = (const T*)t;
        step = 0;
        if constexpr (DMA) {
            base += b * v.b + (long)hk * p.share * v.h;
            step = kStep / p.share * v.l;
        }
        this->open(p.D, v.l, v.h, p.share);
    }
    __device__ __forceinline__ void fetch(const Att& p, const View& v, int b, int hk, unsigned char* to, int st) {
        if constexpr (DMA) {
            const int left = p.R - st * kStep;
            this->load(base + st * step, to, left >= 64 ? ~0ull : (1ull << left) - 1);
        } else {
#pragma unroll
            for (int j = 0; j < L::kPieces; ++j) {
                const int r = st * kStep + L::row(j);
                this->u[j] = make_uint4(0, 0, 0, 0);
                if (r < p.R && L::col(j) < p.D) this->u[j] = *reinterpret_cast<const uint4*>(base + row_at(p, v, b, hk, r) + L::col(j));
            }
        }
    }
};

// this lane's row as the second operand (contracted over the head's width): DP / 16 pieces of 8 elements
template <typename T, int DP>
__device__ __forceinline__ void row_operand(const Att& p, const void* base, const View& v, int b, int hk, int r, bool on,
                                            uint4 (&f)[DP / 16]) {
    const int h = (threadIdx.x & 63) >> 5;
    const T* t = (const T*)base + (on ? row_at(p, v, b, hk, r) : 0);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        const int d = ks * 16 + h * 8;
        f[ks] = make_uint4(0, 0, 0, 0);
        if (on && d < p.D) f[ks] = *reinterpret_cast<const uint4*>(t + d);
    }
}

// In the kernels below no branch stands between a matrix instruction and the first use of its result by an ordinary one:
// where a branch joined again before that use, the compiler counted the wait of the longer way only, and on the shorter
// one the registers were read before they were written.  So results are used first and masks are put in afterwards.

// Every wave's DMA has landed and every wave's reads of the other buffer are done.
__device__ __forceinline__ void arrive() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

struct Work { int b, hk, tile, split; };

// Work item: tiles fastest, then splits, then (image, key head).  Scalars, so that what is addressed with them is too.
__device__ __forceinline__ Work work_of(const Att& p, int tiles) {
    const unsigned id = p.lens ? blockIdx.x : xcd_order(blockIdx.x, gridDim.x), t = id / (unsigned)tiles, bh = t / (unsigned)p.splits;
    Work w;
    w.tile = __builtin_amdgcn_readfirstlane((int)(id - t * (unsigned)tiles));
    w.split = __builtin_amdgcn_readfirstlane((int)(t - bh * (unsigned)p.splits));
    w.b = __builtin_amdgcn_readfirstlane((int)(bh / (unsigned)p.Hk));
    w.hk = __builtin_amdgcn_readfirstlane((int)(bh % (unsigned)p.Hk));
    return w;
}

// Where part s of `blocks` begins (at most 2^23 blocks and 256 parts: the product fits 32 bits, whose division is a tenth of
// a 64-bit one's instructions).
__device__ __forceinline__ int part_of(int blocks, int s, int parts) { return (int)((unsigned)blocks * (unsigned)s / (unsigned)parts); }

// ------------------------------------------------------------------------------------------------ forward
template <typename E, int DP, bool DMA>
__global__ __launch_bounds__(256, DP <= 64 ? 4 : 2) void xa_fwd_kernel(Att p, int tiles) {
    typedef typename E::raw T;
    // (four variables, not an array: the compiler then knows that what is brought into one is not what is read)
    __shared__ __attribute__((aligned(16))) unsigned char K0[Tile<DP>::kBytes], V0[Tile<DP>::kBytes], K1[Tile<DP>::kBytes],
        V1[Tile<DP>::kBytes];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, h = lane >> 5;
    const Work w = work_of(p, tiles);
    const int r = w.tile * kRows + wave * 32 + l31;
    const bool row_on = r < p.R, wave_on = r - l31 < p.R;
    const int len = key_count(p, w.b);
    const int nkb = (len + kKeys - 1) / kKeys;
    const int kb0 = part_of(nkb, w.split, p.splits), kb1 = part_of(nkb, w.split + 1, p.splits);

    uint4 qf[DP / 16];
    row_operand<T, DP>(p, p.q, p.vq, w.b, w.hk, r, row_on, qf);
    f32x16 acc[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) acc[t] = zero16();
    float m = -kInf, l = 0.f;
    const Reads<DP> rd;
    KeyStream<T, DP, DMA> ks_(p, p.k, p.vk, w.b, w.hk), vs_(p, p.v, p.vv, w.b, w.hk);
    KeySets sets(p, w.b, len);
    unsigned long long set = 0, next = 0;
    if (kb0 < kb1) {
        sets.ahead(kb0);
        next = sets.of(kb0);
        ks_.fetch(p, K0, kb0, next);
        vs_.fetch(p, V0, kb0, next);
        sets.ahead(kb0 + 1);
    }
    // one block of keys from (kt, vt), the next on its way into (kn, vn)
    auto block = [&](unsigned char* kt, unsigned char* vt, unsigned char* kn, unsigned char* vn, int kb) {
        if constexpr (!DMA) {
            ks_.put(kt);
            vs_.put(vt);
        }
        set = next;
        arrive();                            // this block has landed; nobody reads (kn, vn) any more
        if (kb + 1 < kb1) {
            next = sets.of(kb + 1);
            ks_.fetch(p, kn, kb + 1, next);
            vs_.fetch(p, vn, kb + 1, next);
            sets.ahead(kb + 2);
        }
        if (!wave_on || set == 0) return;
        // S^T: keys on the registers, this lane's row
        f32x16 st[2] = {zero16(), zero16()};
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
            for (int t = 0; t < 2; ++t) st[t] = E::mfma(rd.rows(kt, t, ks), qf[ks], st[t]);
        float top = row_max(st);
        if (set != ~0ull) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) st[t][i] = key_on(set, t, i) ? st[t][i] : -kInf;
            top = row_max(st);
        }
        top = halves_max(top);
        // The reference m only follows the maximum where it is passed by more than 2^8: probabilities relative to it stay
        // far inside both types' range, and the accumulators are seldom rescaled.  (Without the maximum, the sum of a block's
        // probabilities telling when m no longer serves, the scores have to outlive them: 3 waves a SIMD, A 484 us.)
        if (__any(!(top * p.c <= fmaf(m, p.c, 8.f)))) {
            const float up = __builtin_elementwise_maximum(m, top);
            const float alpha = up == -kInf ? 1.f : __builtin_amdgcn_exp2f((m - up) * p.c);   // (m = -inf: 0)
            l *= alpha;
#pragma unroll
            for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[t][i] *= alpha;
            m = up;
        }
        const float mc = m == -kInf ? 0.f : m * p.c;
        uint4 pf[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            f32x16& x = st[s >> 1];
#pragma unroll
            for (int i = 8 * (s & 1); i < 8 * (s & 1) + 8; ++i) {
                x[i] = __builtin_amdgcn_exp2f(fmaf(x[i], p.c, -mc));
                l += x[i];
            }
            pf[s] = pack_acc<E>(x, s & 1);
        }
        // O^T += V^T P^T
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int t = 0; t < DP / 32; ++t) acc[t] = E::mfma(rd.cols(vt, s, t), pf[s], acc[t]);
    };
    for (int kb = kb0; kb < kb1; kb += 2) {
        block(K0, V0, K1, V1, kb);
        if (kb + 1 < kb1) block(K1, V1, K0, V0, kb + 1);
    }
    const long bh = (long)w.b * p.Hk + w.hk;
    l = halves_sum(l);
    if (!row_on) return;
    if (p.splits > 1) {
        float* o = p.part + ((bh * p.splits + w.split) * p.R + r) * (DP + 2);
        if (h == 0) { o[DP] = m; o[DP + 1] = l; }
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 2)
                *reinterpret_cast<float2*>(o + t * 32 + entry(i, h)) = make_float2(acc[t][i], acc[t][i + 1]);
        return;
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    if (h == 0 && p.lse) p.lse[bh * p.R + r] = log_sum(m, l, p.c);
    T* o = (T*)p.out + dense_row(p, w.b, w.hk, r);
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = t * 32 + 8 * g + 4 * h;
            if (d < p.D) {
                uint2 u;
                u.x = E::pair(acc[t][4 * g] * inv, acc[t][4 * g + 1] * inv);
                u.y = E::pair(acc[t][4 * g + 2] * inv, acc[t][4 * g + 3] * inv);
                *reinterpret_cast<uint2*>(o + d) = u;
            }
        }
}

// Joins the parts of one row: W waves a row, each its range of at most 64 parts, whose statistics it reads in one access and
// whose sums in the next.  One wave for up to 16 parts (33,800 rows of 5 parts of 128 columns: 21 us, 88 MB at 4.2 TB/s), four
// for more.
template <typename E, int DP, int W>
__global__ __launch_bounds__(256) void xa_join_kernel(Att p, unsigned rows) {
    typedef typename E::raw T;
    __shared__ float ms[4], ls[4], as[4][DP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned id = blockIdx.x * (4 / W) + wave / W;
    if (id >= rows) return;                          // (W = 4: a block is a row)
    const unsigned bh = id / (unsigned)p.R, r = id - bh * (unsigned)p.R;
    const int per = (p.splits + W - 1) / W, first = wave % W * per;
    const int mine = p.splits - first < per ? p.splits - first : per;
    const long step = (long)p.R * (DP + 2);
    const float* base = p.part + ((long)bh * p.splits * p.R + r) * (DP + 2) + first * step;
    // lane s weighs part s
    const float own = lane < mine ? base[lane * step + DP] : -kInf, sum = lane < mine ? base[lane * step + DP + 1] : 0.f;
    float m = own;
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) m = __builtin_elementwise_maximum(m, __shfl_xor(m, k, 64));
    const float f = m == -kInf ? 0.f : __builtin_amdgcn_exp2f((own - m) * p.c);
    float l = wave_sum(sum * f);
    float a0 = 0.f, a1 = 0.f;
    const int d = lane * 2;
#pragma unroll 8
    for (int s = 0; s < mine; ++s) {
        const float g = __shfl(f, s, 64);
        if (d < DP) {
            const float2 o = *reinterpret_cast<const float2*>(base + s * step + d);
            a0 = fmaf(o.x, g, a0);
            a1 = fmaf(o.y, g, a1);
        }
    }
    if constexpr (W > 1) {
        if (lane == 0) { ms[wave] = m; ls[wave] = l; }
        if (d < DP) { as[wave][d] = a0; as[wave][d + 1] = a1; }
        __syncthreads();
        if (wave) return;
        m = ms[0];
#pragma unroll
        for (int w = 1; w < W; ++w) m = __builtin_elementwise_maximum(m, ms[w]);
        l = a0 = a1 = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float g = m == -kInf ? 0.f : __builtin_amdgcn_exp2f((ms[w] - m) * p.c);
            l = fmaf(ls[w], g, l);
            if (d < DP) { a0 = fmaf(as[w][d], g, a0); a1 = fmaf(as[w][d + 1], g, a1); }
        }
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    if (lane == 0 && p.lse) p.lse[id] = log_sum(m, l, p.c);
    if (d < p.D) {
        T* o = (T*)p.out + dense_row(p, bh / (unsigned)p.Hk, bh % (unsigned)p.Hk, r);
        *reinterpret_cast<unsigned*>(o + d) = E::pair(a0 * inv, a1 * inv);
    }
}

// ------------------------------------------------------------------------------------------------ backward
// dq of 128 rows, and delta for xa_dkv.  delta = rowsum(do o) comes from the rounded o; over a few keys o is as large as
// v and that rounding would show in dS = P (dP - delta), so an image whose keys lie within one block (its length: a mask may
// leave as few of a longer one) takes delta = sum_j P_j dP_j from its registers instead.
template <typename E, int DP, bool DMA>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : 2) void xa_dq_kernel(Att p, int tiles) {
    typedef typename E::raw T;
    __shared__ __attribute__((aligned(16))) unsigned char K0[Tile<DP>::kBytes], V0[Tile<DP>::kBytes], K1[Tile<DP>::kBytes],
        V1[Tile<DP>::kBytes];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, h = lane >> 5;
    const Work w = work_of(p, tiles);
    const int r = w.tile * kRows + wave * 32 + l31;
    const bool row_on = r < p.R, wave_on = w.tile * kRows + wave * 32 < p.R;
    const int len = key_count(p, w.b);
    const int nkb = (len + kKeys - 1) / kKeys;
    const int kb0 = part_of(nkb, w.split, p.splits), kb1 = part_of(nkb, w.split + 1, p.splits);
    const long bh = (long)w.b * p.Hk + w.hk;

    uint4 qf[DP / 16], df[DP / 16];
    row_operand<T, DP>(p, p.q, p.vq, w.b, w.hk, r, row_on, qf);
    row_operand<T, DP>(p, p.dout, p.vd, w.b, w.hk, r, row_on, df);
    const float lse = row_on ? p.lse[bh * p.R + r] : kInf;
    float del = 0.f;
    if (nkb > 1) {
        uint4 of[DP / 16];
        const View vo = {(long)p.R * p.Hk * p.D, (long)p.share * p.Hk * p.D, p.D};
        row_operand<T, DP>(p, p.o, vo, w.b, w.hk, r, row_on, of);
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
            const unsigned a[4] = {of[ks].x, of[ks].y, of[ks].z, of[ks].w}, c[4] = {df[ks].x, df[ks].y, df[ks].z, df[ks].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float a0, a1, c0, c1;
                E::unpair(a[i], a0, a1);
                E::unpair(c[i], c0, c1);
                del = fmaf(a0, c0, fmaf(a1, c1, del));
            }
        }
        del = halves_sum(del);
        if (w.split == 0 && row_on && h == 0) p.delta[bh * p.R + r] = -del;
    }
    f32x16 acc[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) acc[t] = zero16();

    const Reads<DP> rd;
    KeyStream<T, DP, DMA> ks_(p, p.k, p.vk, w.b, w.hk), vs_(p, p.v, p.vv, w.b, w.hk);
    KeySets sets(p, w.b, len);
    unsigned long long set = 0, next = 0;
    int seen = 0;                                       // keys that take part
    if (kb0 < kb1) {
        sets.ahead(kb0);
        next = sets.of(kb0);
        ks_.fetch(p, K0, kb0, next);
        vs_.fetch(p, V0, kb0, next);
        sets.ahead(kb0 + 1);
    }
    auto block = [&](unsigned char* kt, unsigned char* vt, unsigned char* kn, unsigned char* vn, int kb) {
        if constexpr (!DMA) {
            ks_.put(kt);
            vs_.put(vt);
        }
        set = next;
        seen += __popcll(set);
        arrive();
        if (kb + 1 < kb1) {
            next = sets.of(kb + 1);
            ks_.fetch(p, kn, kb + 1, next);
            vs_.fetch(p, vn, kb + 1, next);
            sets.ahead(kb + 2);
        }
        if (!wave_on || set == 0) return;
        // P (dP - delta) of 32 keys: keys on the registers, this lane's row
        auto scores = [&](int t, f32x16& s) {
            s = zero16();
            f32x16 dp = splat16(-del);
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                s = E::mfma(rd.rows(kt, t, ks), qf[ks], s);
                dp = E::mfma(rd.rows(vt, t, ks), df[ks], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], p.c, -lse)) * dp[i];
            if (set != ~0ull) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = key_on(set, t, i) ? s[i] : 0.f;
            }
        };
        if (nkb == 1) {
            float sum = 0.f;
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
                f32x16 s;
                scores(t, s);
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += s[i];
            }
            del = halves_sum(sum);
            if (row_on && h == 0) p.delta[bh * p.R + r] = -del;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x16 s;
            scores(t, s);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint4 sf = pack_acc<E>(s, k);
#pragma unroll
                for (int u = 0; u < DP / 32; ++u) acc[u] = E::mfma(rd.cols(kt, 2 * t + k, u), sf, acc[u]);
            }
        }
    };
    for (int kb = kb0; kb < kb1; kb += 2) {
        block(K0, V0, K1, V1, kb);
        if (kb + 1 < kb1) block(K1, V1, K0, V0, kb + 1);
    }
    if (seen == 1 && single_key(p, w.b, len)) {
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) acc[t] *= splat16(0.f);
    }
    if (!row_on) return;
    const long at = dense_row(p, w.b, w.hk, r);
    const long whole = (long)p.B * p.Hk * p.R * p.D;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = t * 32 + 8 * g + 4 * h;
            if (d >= p.D) continue;
            if (p.splits > 1) {
                *reinterpret_cast<float4*>(p.part + (long)w.split * whole + at + d) =
                    make_float4(acc[t][4 * g], acc[t][4 * g + 1], acc[t][4 * g + 2], acc[t][4 * g + 3]);
            } else {
                uint2 u;
                u.x = E::pair(acc[t][4 * g] * p.scale, acc[t][4 * g + 1] * p.scale);
                u.y = E::pair(acc[t][4 * g + 2] * p.scale, acc[t][4 * g + 3] * p.scale);
                *reinterpret_cast<uint2*>((T*)p.dq + at + d) = u;
            }
        }
}

// dk and dv of 128 keys.  A key is a column of every product here, so what a masked key's lane computes reaches no other:
// it is thrown away at the end.  Two waves a SIMD up to 96 columns (5 images of 0 to 777 masked keys, 8 heads of 96 on 2,
// fp16: 37 us, 48 with one); at 128 two waves spill 12 registers, which long products repay (4 x 16 heads, 4,000 rows and
// keys: 1,132 us against 1,241) and short ones do not (256 workgroups of 10 steps: 49 against 40): one wave there.
template <typename E, int DP, bool DMA>
__global__ __launch_bounds__(256, DP <= 96 ? 2 : 1) void xa_dkv_kernel(Att p, int tiles) {
    typedef typename E::raw T;
    __shared__ __attribute__((aligned(16))) unsigned char Q0[Tile<DP>::kBytes], D0[Tile<DP>::kBytes], Q1[Tile<DP>::kBytes],
        D1[Tile<DP>::kBytes];
    __shared__ __attribute__((aligned(16))) float S0[2][kStep], S1[2][kStep];        // log of the sum | -delta of the rows
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l31 = lane & 31, h = lane >> 5;
    const Work w = work_of(p, tiles);
    const int key = w.tile * kRows + wave * 32 + l31;
    const int len = key_count(p, w.b);
    bool on = key < len;
    if (on && p.mask) on = p.mask[(long)w.b * p.mask_ld + key] != 0;
    const bool wave_on = __any(on);
    // (here, where every lane of the wave takes part; a key is on two lanes)
    const bool lone = __popcll(__ballot(on)) == 2 && single_key(p, w.b, len);
    const long bh = (long)w.b * p.Hk + w.hk;
    const int nst = (p.R + kStep - 1) / kStep;
    const int st0 = part_of(nst, w.split, p.splits);
    const int st1 = w.tile * kRows < len ? part_of(nst, w.split + 1, p.splits) : st0;

    uint4 kf[DP / 16], vf[DP / 16];
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
        const int d = ks * 16 + h * 8;
        kf[ks] = vf[ks] = make_uint4(0, 0, 0, 0);
        if (on && d < p.D) {
            kf[ks] = *reinterpret_cast<const uint4*>((const T*)p.k + w.b * p.vk.b + w.hk * p.vk.h + key * p.vk.l + d);
            vf[ks] = *reinterpret_cast<const uint4*>((const T*)p.v + w.b * p.vv.b + w.hk * p.vv.h + key * p.vv.l + d);
        }
    }
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) dk[t] = dv[t] = zero16();

    const Reads<DP> rd;
    RowStream<T, DP, DMA> qs(p, p.q, p.vq, w.b, w.hk), ds(p, p.dout, p.vd, w.b, w.hk);
    // Rows beyond the last are zeros everywhere, statistics included: P = 1 there meets zeros of q and dout.
    const __amdgpu_buffer_rsrc_t lse = buffer_at(p.lse + bh * p.R, p.R * 4u), del = buffer_at(p.delta + bh * p.R, p.R * 4u);
    auto fetch = [&](unsigned char* qn, unsigned char* dn, float (*sn)[kStep], int st) {
        qs.fetch(p, p.vq, w.b, w.hk, qn, st);
        ds.fetch(p, p.vd, w.b, w.hk, dn, st);
        const int wv = Tile<DP>::wave();
        if (wv < 2)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wv ? del : lse, (__attribute__((address_space(3))) void*)sn[wv], 4,
                                                     (unsigned)(st * kStep + lane) * 4u, 0, 0, 0);
    };
    if (st0 < st1) fetch(Q0, D0, S0, st0);
    auto block = [&](unsigned char* qt, unsigned char* dt, float (*sv)[kStep], unsigned char* qn, unsigned char* dn,
                     float (*sn)[kStep], int st) {
        if constexpr (!DMA) {
            qs.put(qt);
            ds.put(dt);
        }
        arrive();
        if (st + 1 < st1) fetch(qn, dn, sn, st + 1);
        if (!wave_on) return;
        // two halves of 32 rows
        f32x16 s[2], dp[2];
        uint4 pf[2][2], df[2][2];
        auto products = [&](int u) {                      // S and dP - delta: rows on the registers, this lane's key
            s[u] = zero16();
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 x = *reinterpret_cast<const float4*>(&sv[1][u * 32 + 8 * g + 4 * h]);
                dp[u][4 * g] = x.x; dp[u][4 * g + 1] = x.y; dp[u][4 * g + 2] = x.z; dp[u][4 * g + 3] = x.w;
            }
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                s[u] = E::mfma(rd.rows(qt, u, ks), kf[ks], s[u]);
                dp[u] = E::mfma(rd.rows(dt, u, ks), vf[ks], dp[u]);
            }
        };
        auto probabilities = [&](int u) {                 // P and dS, packed
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 x = *reinterpret_cast<const float4*>(&sv[0][u * 32 + 8 * g + 4 * h]);
                const float lse[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[u][4 * g + i] = __builtin_amdgcn_exp2f(fmaf(s[u][4 * g + i], p.c, -lse[i]));
                    dp[u][4 * g + i] *= s[u][4 * g + i];
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) { pf[u][k] = pack_acc<E>(s[u], k); df[u][k] = pack_acc<E>(dp[u], k); }
        };
        auto gradients = [&](int u) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int t = 0; t < DP / 32; ++t) {
                    dv[t] = E::mfma(rd.cols(dt, 2 * u + k, t), pf[u][k], dv[t]);
                    dk[t] = E::mfma(rd.cols(qt, 2 * u + k, t), df[u][k], dk[t]);
                }
        };
        products(0);
        probabilities(0);
        gradients(0);
        products(1);
        probabilities(1);
        gradients(1);
    };
    for (int st = st0; st < st1; st += 2) {
        block(Q0, D0, S0, Q1, D1, S1, st);
        if (st + 1 < st1) block(Q1, D1, S1, Q0, D0, S0, st + 1);
    }
    if (key >= p.Lk) return;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) {
        if (lone) dk[t] *= splat16(0.f);
        if (!on) dk[t] = dv[t] = zero16();
    }
    const long at = (((long)w.b * p.Lk + key) * p.Hk + w.hk) * p.D;
    const long whole = (long)p.B * p.Lk * p.Hk * p.D;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = t * 32 + 8 * g + 4 * h;
            if (d >= p.D) continue;
            if (p.splits > 1) {
                float* o = p.part + (long)w.split * 2 * whole + at + d;
                *reinterpret_cast<float4*>(o) = make_float4(dk[t][4 * g], dk[t][4 * g + 1], dk[t][4 * g + 2], dk[t][4 * g + 3]);
                *reinterpret_cast<float4*>(o + whole) = make_float4(dv[t][4 * g], dv[t][4 * g + 1], dv[t][4 * g + 2], dv[t][4 * g + 3]);
            } else {
                uint2 u;
                u.x = E::pair(dk[t][4 * g] * p.scale, dk[t][4 * g + 1] * p.scale);
                u.y = E::pair(dk[t][4 * g + 2] * p.scale, dk[t][4 * g + 3] * p.scale);
                *reinterpret_cast<uint2*>((T*)p.dk + at + d) = u;
                u.x = E::pair(dv[t][4 * g], dv[t][4 * g + 1]);
                u.y = E::pair(dv[t][4 * g + 2], dv[t][4 * g + 3]);
                *reinterpret_cast<uint2*>((T*)p.dv + at + d) = u;
            }
        }
}

// One or two arrays (blockIdx.y) of `count` elements: out[i] = factor * sum over parts of part[s][i], four elements a thread;
// a part holds the arrays one behind the other.  A's dk and dv, 4 parts: 160 MB in 25 us
// (6.4 TB/s; they are still in the last level of cache).
template <typename T> struct Sums { T* out[2]; float factor[2]; };

template <typename E>
__global__ __launch_bounds__(256) void xa_sum_kernel(const float* part, int parts, long count, Sums<typename E::raw> to) {
    const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4, stride = gridDim.y * count;
    if (i >= count) return;
    part += blockIdx.y * count + i;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < parts; s += 8) {             // eight parts' loads in flight
        float4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            v[k] = s + k < parts ? *reinterpret_cast<const float4*>(part + (s + k) * stride) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; ++k) { a.x += v[k].x; a.y += v[k].y; a.z += v[k].z; a.w += v[k].w; }
    }
    const float factor = to.factor[blockIdx.y];
    uint2 u;
    u.x = E::pair(a.x * factor, a.y * factor);
    u.y = E::pair(a.z * factor, a.w * factor);
    *reinterpret_cast<uint2*>(to.out[blockIdx.y] + i) = u;
}

int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }

// Parts of a long axis, at most `most` and of two blocks at least: `groups` workgroups of `steps` blocks each run in rounds of
// `slots` workgroups, so the time goes with rounds / parts; each part more costs the join the time of about `extra` blocks.
int parts_for(long groups, long steps, long slots, double extra, long most) {
    if ((steps + 1) / 2 < most) most = (steps + 1) / 2;
    int best = 1;
    double least = 1e300;
    for (long n = 1; n <= most; ++n) {
        const double rounds = (double)((groups * n + slots - 1) / slots);
        const double cost = rounds * (double)((steps + n - 1) / n) + (n > 1 ? extra * (double)n * (double)groups / slots : 0.0);
        if (cost < least * 0.98) { least = cost; best = (int)n; }
    }
    return best;
}

constexpr long kCus = 256;

struct Plan { long row_groups, key_groups; int rtiles, ktiles, fwd, dkv, dq, dp; };

Plan plan_of(int B, long R, int Lk, int Hk, int D) {
    Plan n;
    n.dp = padded(D);
    n.rtiles = (int)((R + kRows - 1) / kRows);
    n.ktiles = (Lk + kRows - 1) / kRows;
    n.row_groups = (long)B * Hk * n.rtiles;
    n.key_groups = (long)B * Hk * n.ktiles;
    // workgroups that a CU holds: registers for heads of 96 and more, LDS and registers for the rest
    const long keys = (Lk + kKeys - 1) / kKeys, rows = (R + kStep - 1) / kStep;
    // (what a join costs goes with the rows or keys that a tile really has)
    const double rowjoin = 6.0 * (double)(R < kRows ? R : kRows) / kRows, keyjoin = 6.0 * (double)(Lk < kRows ? Lk : kRows) / kRows;
    n.fwd = parts_for(n.row_groups, keys, (n.dp <= 64 ? 4 : 2) * kCus, rowjoin, 256);
    n.dq = parts_for(n.row_groups, keys, (n.dp <= 64 ? 3 : 2) * kCus, rowjoin, 64);
    n.dkv = parts_for(n.key_groups, rows, (n.dp <= 64 ? 3 : n.dp <= 96 ? 2 : 1) * kCus, keyjoin, 64);
    return n;
}

bool bad(int B, int Lq, int Lk, int Hk, int share, int D) {
    return B <= 0 || Lq <= 0 || Lk <= 0 || Hk <= 0 || share <= 0 || D <= 0 || D % 8 || D > 128 ||
           (long)Lq * share > (1L << 29) || (long)B * Hk * share > 0x7fffffffL || Lk > (1 << 29);
}

bool bad_grid(long n) { return n <= 0 || n > 0x7fffffffL; }

// A tile's rows lie within 31 bits of its first (DMA offsets).
bool near(long a, long b) { return a < (1L << 23) && b < (1L << 23); }
bool near_keys(const Att& p) { return near(p.vk.l, p.vv.l); }
bool near_rows(const Att& p) {
    return kStep % p.share == 0 && near(p.vq.l, p.vd.l) && near(p.vq.h * p.share / kStep, p.vd.h * p.share / kStep);
}

template <typename E, int DP> int launch_fwd(Att p, const Plan& n, hipStream_t st) {
    p.splits = n.fwd;
    const long blocks = n.row_groups * n.fwd, rows = (long)p.B * p.Hk * p.R;
    if (bad_grid(blocks) || (n.fwd > 1 && bad_grid(rows))) return -3;
    const auto kernel = near_keys(p) ? xa_fwd_kernel<E, DP, true> : xa_fwd_kernel<E, DP, false>;
    kernel<<<dim3((unsigned)blocks), 256, 0, st>>>(p, n.rtiles);
    if (n.fwd > 16) xa_join_kernel<E, DP, 4><<<dim3((unsigned)rows), 256, 0, st>>>(p, (unsigned)rows);
    else if (n.fwd > 1) xa_join_kernel<E, DP, 1><<<dim3((unsigned)((rows + 3) / 4)), 256, 0, st>>>(p, (unsigned)rows);
    return DP_LAUNCH_STATUS();
}

template <typename E, int DP> int launch_bwd(Att p, const Plan& n, hipStream_t st) {
    typedef typename E::raw T;
    const long kv = (long)p.B * p.Lk * p.Hk * p.D, qn = (long)p.B * p.Hk * p.R * p.D;
    if (bad_grid(n.key_groups * n.dkv) || bad_grid(n.row_groups * n.dq) || bad_grid((kv + 1023) / 1024) ||
        bad_grid((qn + 1023) / 1024))
        return -3;
    p.splits = n.dq;
    const auto dq = near_keys(p) ? xa_dq_kernel<E, DP, true> : xa_dq_kernel<E, DP, false>;
    const auto dkv = near_rows(p) ? xa_dkv_kernel<E, DP, true> : xa_dkv_kernel<E, DP, false>;
    dq<<<dim3((unsigned)(n.row_groups * n.dq)), 256, 0, st>>>(p, n.rtiles);
    if (n.dq > 1)
        xa_sum_kernel<E><<<dim3((unsigned)((qn + 1023) / 1024)), 256, 0, st>>>(p.part, n.dq, qn, {{(T*)p.dq, nullptr}, {p.scale, 1.f}});
    p.splits = n.dkv;
    dkv<<<dim3((unsigned)(n.key_groups * n.dkv)), 256, 0, st>>>(p, n.ktiles);
    if (n.dkv > 1)
        xa_sum_kernel<E><<<dim3((unsigned)((kv + 1023) / 1024), 2), 256, 0, st>>>(p.part, n.dkv, kv,
                                                                                   {{(T*)p.dk, (T*)p.dv}, {p.scale, 1.f}});
    return DP_LAUNCH_STATUS();
}

template <template <typename, int> class Run> int dispatch(int fp16, int dp, const Att& p, const Plan& n, hipStream_t st) {
    switch (dp + fp16) {
        case 32: return Run<Bf, 32>::go(p, n, st);
        case 33: return Run<Hf, 32>::go(p, n, st);
        case 64: return Run<Bf, 64>::go(p, n, st);
        case 65: return Run<Hf, 64>::go(p, n, st);
        case 96: return Run<Bf, 96>::go(p, n, st);
        case 97: return Run<Hf, 96>::go(p, n, st);
        case 128: return Run<Bf, 128>::go(p, n, st);
        case 129: return Run<Hf, 128>::go(p, n, st);
    }
    return -1;
}

template <typename E, int DP> struct RunFwd {
    static int go(const Att& p, const Plan& n, hipStream_t st) { return launch_fwd<E, DP>(p, n, st); }
};
template <typename E, int DP> struct RunBwd {
    static int go(const Att& p, const Plan& n, hipStream_t st) { return launch_bwd<E, DP>(p, n, st); }
};

bool misaligned(const void* p, const long* s) { return ((uintptr_t)p & 15) || s[0] % 8 || s[1] % 8 || s[2] % 8; }

}  // namespace

// floats of workspace for the parts of split axes (0: none); backward's covers dk and dv, then dq
DP_EXPORT long dp_xa_workspace(int B, int Lq, int Lk, int Hk, int share, int D, int backward) {
    if (bad(B, Lq, Lk, Hk, share, D)) return -1;
    const long R = (long)Lq * share;
    const Plan n = plan_of(B, R, Lk, Hk, D);
    if (!backward) return n.fwd > 1 ? (long)B * Hk * n.fwd * R * (n.dp + 2) : 0;
    const long a = n.dkv > 1 ? 2L * n.dkv * B * Lk * Hk * D : 0, b = n.dq > 1 ? (long)n.dq * B * Hk * R * D : 0;
    return a > b ? a : b;
}

// strides: image, position and head of q, k and v (nine), in elements
DP_EXPORT int dp_xa_fwd(const void* q, const void* k, const void* v, void* out, float* lse, const int* lens,
                        const void* mask, long mask_ld, float* ws, const long* strides, int B, int Lq, int Lk, int Hk,
                        int share, int D, float scale, int fp16, void* stream) {
    if (bad(B, Lq, Lk, Hk, share, D) || !q || !k || !v || !out || !strides || misaligned(q, strides) ||
        misaligned(k, strides + 3) || misaligned(v, strides + 6) || ((uintptr_t)out & 15) || !(scale > 0.f))
        return -2;
    Att p{};
    p.q = q; p.k = k; p.v = v; p.out = out; p.lse = lse; p.lens = lens; p.mask = (const unsigned char*)mask; p.mask_ld = mask_ld;
    p.vq = {strides[0], strides[1], strides[2]}; p.vk = {strides[3], strides[4], strides[5]};
    p.vv = {strides[6], strides[7], strides[8]};
    p.B = B; p.Lq = Lq; p.Lk = Lk; p.Hk = Hk; p.share = share; p.D = D; p.R = Lq * share;
    p.scale = scale; p.c = scale * 1.4426950408889634f; p.part = ws;
    const Plan n = plan_of(B, p.R, Lk, Hk, D);
    if (n.fwd > 1 && !ws) return -2;
    return dispatch<RunFwd>(fp16, n.dp, p, n, (hipStream_t)stream);
}

// strides: image, position and head of q, k, v and dout (twelve); o and the gradients are dense; delta: scratch like lse
DP_EXPORT int dp_xa_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout, const float* lse,
                        float* delta, void* dq, void* dk, void* dv, const int* lens, const void* mask, long mask_ld,
                        float* ws, const long* strides, int B, int Lq, int Lk, int Hk, int share, int D, float scale,
                        int fp16, void* stream) {
    if (bad(B, Lq, Lk, Hk, share, D) || !q || !k || !v || !o || !dout || !lse || !delta || !dq || !dk || !dv || !strides ||
        misaligned(q, strides) || misaligned(k, strides + 3) || misaligned(v, strides + 6) || misaligned(dout, strides + 9) ||
        (((uintptr_t)o | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) || !(scale > 0.f))
        return -2;
    Att p{};
    p.q = q; p.k = k; p.v = v; p.o = o; p.dout = dout; p.lse = const_cast<float*>(lse); p.delta = delta;
    p.dq = dq; p.dk = dk; p.dv = dv; p.lens = lens; p.mask = (const unsigned char*)mask; p.mask_ld = mask_ld;
    p.vq = {strides[0], strides[1], strides[2]}; p.vk = {strides[3], strides[4], strides[5]};
    p.vv = {strides[6], strides[7], strides[8]}; p.vd = {strides[9], strides[10], strides[11]};
    p.B = B; p.Lq = Lq; p.Lk = Lk; p.Hk = Hk; p.share = share; p.D = D; p.R = Lq * share;
    p.scale = scale; p.c = scale * 1.4426950408889634f; p.part = ws;
    const Plan n = plan_of(B, p.R, Lk, Hk, D);
    if ((n.dkv > 1 || n.dq > 1) && !ws) return -2;
    return dispatch<RunBwd>(fp16, n.dp, p, n, (hipStream_t)stream);
}
