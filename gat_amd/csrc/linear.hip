// Linear layer with its epilogue:  y = act(x W^T + b) + residual,  and its gradient
//     dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz   (d residual = dy)
// on the matrix cores, in f32, bf16 or f16; every sum is kept in f32.
//
//  * 16-bit tensors multiply as they are (v_mfma_f32_32x32x16_{bf16,f16}).
//  * f32 tensors are cut into three bf16 pieces each, v = p0 + p1 + p2, and multiply as the
//    six products p_i q_j with i + j <= 2: what is left out is 2^-25 of a product, less than an f32
//    multiply rounds, at 16/6 of the f32 MFMA's rate.  The pieces are exact for |v| from 2^-110 (7.7e-34) on; of a
//    smaller v they hold the nearest multiple of bf16's smallest number, 2^-133 (the matrix cores keep subnormals).
//    A sum that comes out infinite or NaN (an operand was, or a piece rounded up to infinity next to the largest
//    float) is taken again in plain f32.
//  * act'(z) is written by the forward when a backward follows: f32 for f32 tensors, for 16-bit ones in 16 bits, to
//    2^-16 and, where a unit is saturated and the slope small, to 2^-11 of itself (see pack_slope).
//  * dz = dy act'(z) of 16-bit tensors does not fit their type.  It enters the products as two numbers of it,
//    dz = hi + lo, lo what hi's rounding left: a product more a step, and dx and dW are rounded once, as they
//    are stored.  (One number: every dz off by up to half a step, and the error of dx and dW larger by sqrt 2.)
//    ReLU's slopes are 0 and 1, dz is dy or nothing, and one number is enough.  An infinite or NaN factor on the
//    other side would meet a lo of zero, or of the other sign than hi: such sums are made with hi for lo, twice the
//    sum of the rounded dz (dx: where lin_image_kernel has seen such weights; dW: in a second pass, see `redo`).
//
// What bounds it (times of the kernels alone under the profiler, whose clock varies by a few percent from run to run).
// The forward of layers of a few hundred columns is bound by memory for 16-bit types: [2449029, 256] x [256, 256] bf16
// with GELU and residual takes 1.14 ms (5.0 GB, 4.4 TB/s), where a copy runs at 4.9 TB/s.  Its gradients carry two
// products for one and the slope's decoding: dx 1.01 ms (3.8 GB, 3.7 TB/s), dW 1.14 ms (3.8 GB, 3.3 TB/s; with dz in one
// number they took 0.85 and 0.71).  Wide layers are bound by what feeds the matrix cores: [65537, 1024] x [1024, 1001]
// f16 in 0.177 ms, 760 TFLOP/s, with the matrix cores, LDS and the vector units busy for a third of it each.  f32 is
// between the two: [100000, 240] x [240, 240] takes 0.145 ms forward, of which the matrix cores are busy for 0.031, the
// vector units (cutting the operands, the activation) for 0.037, and 384 MB at the copy's rate are 0.078; dx 0.124, dW
// 0.105.  Launched one behind the other the three take 0.36 ms.
#include "attn_device.h"
#include "common.h"
#include "dense_device.h"

namespace gatmi {

typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));
typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes from any element on

// act'(z), in -0.129 .. 1.129, in 16 bits.  Codes from kSlopeLin on are fixed point of step 2^-15, so that a sum of
// slopes near 1 loses nothing to speak of.  The codes below are a floating-point number of 1024 codes an octave, for
// slopes of the sign that the activation's lower tail has (ELU's is positive, SiLU's and GELU's negative) and below
// 2^-5: a saturated unit's, down to 2^-27 (z = -18 of ELU) to eleven bits, and in steps of 2^-37 from there.  0 and 1
// are exact, 65535 stands for NaN.
constexpr uint32_t kSlopeLin = 23 * 1024, kSlopeZero = kSlopeLin + 4300;     // 4300 steps: 0.1312
constexpr float kSlopeScale = 0x1p99f;                                       // kSlopeLin << 13, as a float, times the scale: 2^-5
constexpr uint32_t kMagic = 0x4b000000u;                                     // 2^23: the integers from there on end a float's bits
constexpr bool slope_tail_negative(int act) { return act == GATMI_ACT_SILU || act == GATMI_ACT_GELU; }
template <bool NEGATIVE> __device__ __forceinline__ uint16_t pack_slope(float d) {
    // of the other sign, 2^-5 or more (once rounded) or NaN: kSlopeLin or more
    const uint32_t small = (__float_as_uint((NEGATIVE ? -d : d) * (1.0f / kSlopeScale)) + 0x1000u) >> 13;
    // v_med3 takes the least of the others for a NaN: the last code
    constexpr float least = -(65535.f - kSlopeZero) / 32768.f;
    const float t = __builtin_amdgcn_fmed3f(-d, least, 0.1312f);
    const uint32_t lin = __float_as_uint(fmaf(t, -32768.f, 8388608.f + kSlopeZero));
    return (uint16_t)(small < kSlopeLin ? small : lin);
}
// scale: kSlopeScale with the tail's sign.  (65535 is left to the caller.)
__device__ __forceinline__ float unpack_slope(uint32_t code, float scale) {
    const uint32_t c = kMagic | code;
    const float lin = fmaf(__uint_as_float(c), 1.0f / 32768.f, -(8388608.f + kSlopeZero) / 32768.f);
    const float small = __uint_as_float(c << 13) * scale;          // (kMagic's bits leave at the top)
    return c < kMagic + kSlopeLin ? small : lin;
}
template <class T> struct SlopeOf { typedef uint16_t type; };
template <> struct SlopeOf<float> { typedef float type; };
template <class T, int ACT> __device__ __forceinline__ typename SlopeOf<T>::type slope_out(float d) {
    if constexpr (IsF32<T>::value) return d;
    else return pack_slope<slope_tail_negative(ACT)>(d);
}

// What the kernels need to know of an element type
template <class T> struct Mul;
template <> struct Mul<bf16_t> {
    static constexpr int PIECES = 1, BK = 64;
    static __device__ __forceinline__ f32x16v mma(u32x4 a, u32x4 b, f32x16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0, 0, 0);
    }
};
template <> struct Mul<f16_t> {
    static constexpr int PIECES = 1, BK = 64;
    static __device__ __forceinline__ f32x16v mma(u32x4 a, u32x4 b, f32x16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8v, a), __builtin_bit_cast(f16x8v, b), c, 0, 0, 0);
    }
};
template <> struct Mul<float> {
    static constexpr int PIECES = 3, BK = 32;
    static __device__ __forceinline__ f32x16v mma(u32x4 a, u32x4 b, f32x16v c) { return Mul<bf16_t>::mma(a, b, c); }
};

// Eight consecutive elements of a row as they lie in memory.  The loads of the main loops have no branch
// around them -- a load under a condition is waited for where the paths join, not where it is used -- so a
// granule that would run over the end of its row starts at the row's last eight elements instead and `drop`
// zeroes, on the way into LDS, the ones that belong to the granule before it.
template <class T> struct Gran {
    uint32_t w[2 * sizeof(T)];
};
template <class T> __device__ __forceinline__ Gran<T> ld_gran(const void *base, uint32_t bytes) {
    Gran<T> g;
    const u32x4u *p = reinterpret_cast<const u32x4u *>(static_cast<const char *>(base) + bytes);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const u32x4u v = p[i];
        g.w[4 * i] = v[0]; g.w[4 * i + 1] = v[1]; g.w[4 * i + 2] = v[2]; g.w[4 * i + 3] = v[3];
    }
    return g;
}
// rows of fewer than eight elements: `left` of them exist
template <class T> __device__ __forceinline__ Gran<T> ld_gran_short(const void *base, uint32_t bytes, int left) {
    Gran<T> g;
    const T *p = reinterpret_cast<const T *>(static_cast<const char *>(base) + bytes);
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < left ? p[i] : (T)0.f;
    __builtin_memcpy(g.w, e, sizeof(e));
    return g;
}
template <class T> __device__ __forceinline__ void drop(Gran<T> &g, int first) {
#pragma unroll
    for (int i = 0; i < (int)(2 * sizeof(T)); ++i) {
        if constexpr (sizeof(T) == 4) g.w[i] = i < first ? 0u : g.w[i];
        else g.w[i] &= 2 * i + 1 < first ? 0u : (2 * i < first ? 0xffff0000u : 0xffffffffu);
    }
}

// A granule that was loaded `over` elements early, moved to its place; zeros follow
template <class T> __device__ __forceinline__ void shift_down(uint32_t (&w)[2 * sizeof(T)], int over) {
    constexpr int W = 2 * sizeof(T);
    if constexpr (sizeof(T) == 2)
        if (over & 1)
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = (w[i] >> 16) | (i + 1 < W ? w[i + 1 < W ? i + 1 : i] << 16 : 0u);
#pragma unroll
    for (int b = sizeof(T) == 2 ? 2 : 1; b < 8; b <<= 1) {
        const int by = sizeof(T) == 2 ? b / 2 : b;
        if (over & b)
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = i + by < W ? w[i + by < W ? i + by : i] : 0u;
    }
    if (over >= 8)
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0u;
}

// (a, b) -> the pair's three bf16 pieces, low half first
__device__ __forceinline__ void cut3(float a, float b, uint32_t &p0, uint32_t &p1, uint32_t &p2) {
    p0 = pack_bf16(a, b);
    a -= __uint_as_float(p0 << 16);
    b -= __uint_as_float(p0 & 0xffff0000u);
    p1 = pack_bf16(a, b);
    a -= __uint_as_float(p1 << 16);
    b -= __uint_as_float(p1 & 0xffff0000u);
    p2 = pack_bf16(a, b);
}

// the eight values of a granule in f32
template <class T> __device__ __forceinline__ VecF<8> gran_values(const Gran<T> &g) {
    VecF<8> v;
    T e[8];
    __builtin_memcpy(e, g.w, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) v.e[i] = (float)e[i];
    return v;
}
template <class T> __device__ __forceinline__ Gran<T> to_gran(const VecF<8> &v) {
    Gran<T> g;
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = (T)v.e[i];
    __builtin_memcpy(g.w, e, sizeof(e));
    return g;
}

// v = hi + lo, both of the tensor's type.  hi stays finite, so that lo is v - hi for every v: infinite where v is
// (v_med3), NaN where v is.  twice: hi again for a finite lo.
template <class T> __device__ __forceinline__ void split2(const VecF<8> &v, Gran<T> &hi, Gran<T> &lo, bool twice) {
    const float top = std::is_same<T, f16_t>::value ? 65504.f : 3.3895313892515355e38f;
    VecF<8> h, l;
#pragma unroll
    for (int i = 0; i < 8; ++i) h.e[i] = __builtin_amdgcn_fmed3f(v.e[i], -top, top);
    hi = to_gran<T>(h);
    h = gran_values<T>(hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) l.e[i] = v.e[i] - h.e[i];
    if (twice)
#pragma unroll
        for (int i = 0; i < 8; ++i) l.e[i] = fabsf(l.e[i]) < INFINITY ? h.e[i] : l.e[i];
    lo = to_gran<T>(l);
}

// A tile of R rows x BK contraction elements in LDS, PIECES planes of 16-bit elements.  16-byte granules
// are XOR-swizzled so that sixteen lanes reading one granule column of sixteen rows hit all 64 banks: rows of
// 128 bytes lie in halves of the banks by their parity, rows of 64 bytes in quarters.
template <class T, int R, int PIECES = Mul<T>::PIECES> struct Tile {
    static constexpr int BK = Mul<T>::BK, G = BK / 8, P = PIECES;
    static constexpr int PLANE = R * BK * 2, BYTES = PLANE * P;
    static __device__ __forceinline__ int at(int row, int g) {
        const int s = G == 8 ? ((row >> 1) & 7) : ((row >> 2) & 3);
        return row * (BK * 2) + ((g ^ s) << 4);
    }
    static __device__ __forceinline__ void put(char *lds, int row, int g, const Gran<T> &v) {
        if constexpr (P == 1) {
            *reinterpret_cast<u32x4 *>(lds + at(row, g)) = u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
        } else {
            uint32_t q[3][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                cut3(__uint_as_float(v.w[2 * i]), __uint_as_float(v.w[2 * i + 1]), q[0][i], q[1][i], q[2][i]);
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<u32x4 *>(lds + p * PLANE + at(row, g)) = u32x4{q[p][0], q[p][1], q[p][2], q[p][3]};
        }
    }
    static __device__ __forceinline__ void put2(char *lds, int row, int g, const VecF<8> &v, bool twice) {
        static_assert(P == 2, "a tile of halves");
        Gran<T> q[2];
        split2<T>(v, q[0], q[1], twice);
#pragma unroll
        for (int p = 0; p < 2; ++p)
            *reinterpret_cast<u32x4 *>(lds + p * PLANE + at(row, g)) = u32x4{q[p].w[0], q[p].w[1], q[p].w[2], q[p].w[3]};
    }
    static __device__ __forceinline__ u32x4 frag(const char *lds, int p, int row, int g) {
        return *reinterpret_cast<const u32x4 *>(lds + p * PLANE + at(row, g));
    }
};

constexpr int kBM = 128;      // rows of dW's tiles

struct LinArgs {
    const void *A, *B;        // [M, K] and [N, K], rows of K elements (B: of ldb)
    const void *plain;        // f32: the weights as they are ([N, K], or [K, N] when A is dy)
    const void *aslope;       // A is multiplied by this slope on its way in (dz = dy act'(z))
    const uint8_t *bad;       // TWO: [rows of B / 32][bad_cols], whether 32 x 32 of B are all finite (0) or not
    int bad_cols;
    const void *bias, *res;
    void *C;                  // [M, N]
    void *slope;              // forward: act'(z) out
    float slope_scale;        // backward: of the slope's coding
    float *part, *dbpart;     // dW: [splits][N][K] slabs, [splits][N] column sums
    void *dw, *db;            // one split: the gradients themselves instead
    long long M;
    int N, K, ldb, act;
    long long tiles_n, tiles;
    long long per_split;      // dW: rows of one split
    int splits;               // dW: of the rows; PART: of the contraction, in pieces of k_split
    int k_split;
};

// Granule of A as it enters the products: dy * slope, rounded to the tensor's type
template <class T> struct SlopeGran {
    uint32_t w[2 * sizeof(T)];
};
template <class T> __device__ __forceinline__ SlopeGran<T> ld_slope(const void *base, uint32_t bytes) {
    SlopeGran<T> s;
    const u32x4u *p = reinterpret_cast<const u32x4u *>(static_cast<const char *>(base) + bytes);
#pragma unroll
    for (int i = 0; i < (int)sizeof(typename SlopeOf<T>::type) / 2; ++i) {
        const u32x4u v = p[i];
        s.w[4 * i] = v[0]; s.w[4 * i + 1] = v[1]; s.w[4 * i + 2] = v[2]; s.w[4 * i + 3] = v[3];
    }
    return s;
}
template <class T> __device__ __forceinline__ SlopeGran<T> ld_slope_short(const void *base, uint32_t bytes, int left) {
    typedef typename SlopeOf<T>::type ST;
    SlopeGran<T> s;
    const ST *p = reinterpret_cast<const ST *>(static_cast<const char *>(base) + bytes);
    ST e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < left ? p[i] : (ST)0;
    __builtin_memcpy(s.w, e, sizeof(e));
    return s;
}
template <class T> __device__ __forceinline__ VecF<8> with_slope(const Gran<T> &g, const SlopeGran<T> &s, float scale) {
    VecF<8> v = gran_values<T>(g);
    if constexpr (IsF32<T>::value) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.e[i] *= __uint_as_float(s.w[i]);
    } else {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 top = __builtin_bit_cast(u16x2, s.w[0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, s.w[i]));
            v.e[2 * i] *= unpack_slope(s.w[i] & 0xffffu, scale);
            v.e[2 * i + 1] *= unpack_slope(s.w[i] >> 16, scale);
        }
        if (top[0] == 65535 || top[1] == 65535)      // a NaN among the eight
            for (int i = 0; i < 8; ++i)
                if (((s.w[i / 2] >> (16 * (i & 1))) & 0xffffu) == 65535u) v.e[i] = __uint_as_float(0x7fc00000u);
    }
    return v;
}

// acc (32x32 blocks of a wave) += one contraction step of 16, all pieces
template <class T, int PA, int MI, int NI>
__device__ __forceinline__ void mma_pieces(const u32x4 (&a)[MI][PA], const u32x4 (&b)[NI][Mul<T>::PIECES],
                                           f32x16v (&acc)[MI][NI]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            if constexpr (Mul<T>::PIECES == 1) {
                if constexpr (PA == 2) acc[i][j] = Mul<T>::mma(a[i][1], b[j][0], acc[i][j]);
                acc[i][j] = Mul<T>::mma(a[i][0], b[j][0], acc[i][j]);
            } else {   // the small products first
                acc[i][j] = Mul<T>::mma(a[i][0], b[j][2], acc[i][j]);
                acc[i][j] = Mul<T>::mma(a[i][2], b[j][0], acc[i][j]);
                acc[i][j] = Mul<T>::mma(a[i][1], b[j][1], acc[i][j]);
                acc[i][j] = Mul<T>::mma(a[i][0], b[j][1], acc[i][j]);
                acc[i][j] = Mul<T>::mma(a[i][1], b[j][0], acc[i][j]);
                acc[i][j] = Mul<T>::mma(a[i][0], b[j][0], acc[i][j]);
            }
        }
}

// acc += A-tile rows ra.. x B-tile rows rb..
template <class T, class TA, class TB, int MI, int NI>
__device__ __forceinline__ void tile_mma(const char *la, const char *lb, int ra, int rb, int lane,
                                         f32x16v (&acc)[MI][NI]) {
    const int r = lane & 31, half = lane >> 5;
    // (two numbers of f16, unrolled whole: registers go to scratch memory)
    constexpr int kUnroll = std::is_same<T, f16_t>::value && TA::P == 2 ? 2 : TA::BK / 16;
#pragma unroll kUnroll
    for (int s = 0; s < TA::BK / 16; ++s) {
        u32x4 a[MI][TA::P], b[NI][TB::P];
#pragma unroll
        for (int p = 0; p < TA::P; ++p) {
#pragma unroll
            for (int i = 0; i < MI; ++i) a[i][p] = TA::frag(la, p, ra + i * 32 + r, 2 * s + half);
            if (p >= TB::P) continue;
#pragma unroll
            for (int j = 0; j < NI; ++j) b[j][p] = TB::frag(lb, p, rb + j * 32 + r, 2 * s + half);
        }
        mma_pieces<T, TA::P, MI, NI>(a, b, acc);
    }
}

// row of accumulator register q in a 32 x 32 block (its column is lane & 31)
__device__ __forceinline__ int acc_row(int q, int half) { return (q >> 2) * 8 + half * 4 + (q & 3); }

// eight columns of one row on their way out: bias, activation, residual, slope
template <class T, int ACT> __device__ __forceinline__ void epi_values(float (&v)[8], const VecF<8> &bias,
                                                                     typename SlopeOf<T>::type (&sl)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        float d;
        v[k] = act_both<ACT, IsF32<T>::value>(v[k] + bias.e[k], d);
        sl[k] = slope_out<T, ACT>(d);
    }
}
template <class T, bool FWD>
__device__ __forceinline__ void epi_piece(const LinArgs &A, long long m, int n, int have, float (&v)[8],
                                          const Gran<T> &bias, const Gran<T> &res) {
    typedef typename SlopeOf<T>::type ST;
    const long long at = m * A.N + n;
    T *out = static_cast<T *>(A.C) + at;
    ST sl[8];
    if constexpr (FWD) {
        GATMI_WITH_ACT(A.act, epi_values<T, ACT>(v, gran_values<T>(bias), sl));
        if (A.slope) {
            ST *so = static_cast<ST *>(A.slope) + at;
            if (have >= 8) {
#pragma unroll
                for (int w = 0; w < (int)sizeof(ST) / 2; ++w) {
                    u32x4u t;
                    __builtin_memcpy(&t, sl + w * (16 / sizeof(ST)), 16);
                    reinterpret_cast<u32x4u *>(so)[w] = t;
                }
            } else {
                for (int k = 0; k < 8; ++k)
                    if (k < have) so[k] = sl[k];
            }
        }
        if (A.res) {
            const VecF<8> rr = gran_values<T>(res);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] += rr.e[k];
        }
    }
    if (have >= 8) {
        VecF<8> o;
#pragma unroll
        for (int k = 0; k < 8; ++k) o.e[k] = v[k];
        stv<T, 8>(out, o);
    } else {
        for (int k = 0; k < 8; ++k)
            if (k < have) out[k] = (T)v[k];
    }
}

// the sum in plain f32, an element at a time: what the pieces cannot say (f32 only)
template <bool FWD> __device__ __forceinline__ float plain_dot(const LinArgs &A, long long m, int n) {
    const float *a = static_cast<const float *>(A.A) + m * A.K;
    const float *sl = FWD || !A.aslope ? nullptr : static_cast<const float *>(A.aslope) + m * A.K;
    const float *w = static_cast<const float *>(A.plain) + (FWD ? (long long)n * A.K : n);
    const long long step = FWD ? 1 : A.N;
    float s = 0.f;
#pragma unroll 1
    for (int k = 0; k < A.K; ++k) s = fmaf(sl ? a[k] * sl[k] : a[k], w[k * step], s);
    return s;
}

// One block a tile, through registers into one LDS buffer: the next step's loads are on their way while this
// one multiplies, and three (f32, backward) or four blocks a CU fill each other's gaps.  128 x 128 by four waves,
// 64 x 64 each, is the largest tile that leaves that many.  Measured without a gain: 128 x 256, 64-row tiles, two
// steps' loads in flight, fragments read a step ahead, wave priorities, partial rows first.
//
// C[m][n] = epilogue(sum_k A[m][k] B[n][k]).  FWD: bias, activation, residual, slope; else A = dy * aslope
// when given.  CUT (f32): B comes as three planes of bf16 pieces, rows of ldb (a multiple of 8, zeros behind K).
// SHORT: K < 8; SHORT_N: N < 8.  PART: a block takes one piece of the contraction and leaves its sums in
// part [splits][M][N], for lin_join_kernel.  WHOLE: K is a multiple of a step, and the last tile of rows starts
// early instead of running over (M >= BM; what it shares with the tile before, that one stores): no address but
// B's rows needs vector arithmetic in the loop, and nothing is dropped.  16-bit types gain 3 to 8% ([65536, 1024] x
// [1024, 1024] bf16 206 -> 192 us); f32, busy with its cuts, loses 2.  TWO (16 bits, backward): dz as two numbers.
template <class T, int BM, int BN, int WM, int WN, bool FWD, bool CUT, bool SHORT, bool SHORT_N, bool PART, bool WHOLE, bool TWO>
__global__ __launch_bounds__(WM * WN * 64, FWD && !IsF32<T>::value ? 4 : 3) void lin_nt_kernel(const LinArgs A) {
    static_assert(!TWO || (!FWD && !IsF32<T>::value), "dz of 16-bit tensors");
    typedef Tile<T, BM, TWO ? 2 : Mul<T>::PIECES> TA;
    typedef Tile<T, BN> TB;
    constexpr int THREADS = WM * WN * 64, MI = BM / WM / 32, NI = BN / WN / 32;
    constexpr int LD = NI * 32 + 4;
    constexpr int kLoop = TA::BYTES + TB::BYTES, kEpi = WM * WN * 16 * LD * 4;
    __shared__ __attribute__((aligned(16))) char smem[kLoop > kEpi ? kLoop : kEpi];
    char *la = smem, *lb = smem + TA::BYTES;
    // consecutive tiles share rows of A: give each XCD (block index mod 8) a contiguous range of them
    const long long item = (long long)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (item >= (PART ? A.tiles * A.splits : A.tiles)) return;
    const long long split = PART ? item / A.tiles : 0, tile = item - split * A.tiles;
    const int k_first = PART ? (int)split * A.k_split : 0;
    const int k_end = PART && k_first + A.k_split < A.K ? k_first + A.k_split : A.K;
    const long long m_first = tile / A.tiles_n * BM, m0 = WHOLE && m_first > A.M - BM ? A.M - BM : m_first;
    const int n0 = (int)(tile % A.tiles_n) * BN;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave / WN) * (MI * 32), wn = (wave % WN) * (NI * 32);
    constexpr int G = TA::G, RP = THREADS / G, NA = BM / RP, NB = (BN + RP - 1) / RP;
    static_assert(BM % RP == 0 && (BN % RP == 0 || BN < RP), "whole tiles a pass");
    typedef typename SlopeOf<T>::type ST;
    Gran<T> ga[NA];
    SlopeGran<T> gs[FWD ? 1 : NA];
    Gran<T> gb[CUT ? 1 : NB];
    u32x4 gc[CUT ? NB : 1][3];
    const int g = threadIdx.x % G, row = threadIdx.x / G;
    const bool sloped = TWO || (!FWD && A.aslope);
    // wave-uniform tile bases, 32-bit offsets from there (a tile spans at most 256 rows of 256 KB); rows behind
    // the matrix repeat its last one, their results are not stored
    const T *ba = static_cast<const T *>(A.A) + m0 * A.K;
    const ST *bs = static_cast<const ST *>(A.aslope) + m0 * A.K;
    const char *bb = static_cast<const char *>(A.B) + (long long)n0 * A.ldb * (CUT ? 2 : (int)sizeof(T));
    const long long plane = (long long)A.N * A.ldb * 2;
    const int left_a = A.M - 1 - m0 < BM ? (int)(A.M - 1 - m0) : BM, left_b = A.N - 1 - n0;
    const int last = CUT ? A.ldb - 8 : A.K - 8;     // B's last whole granule
    // WHOLE: no granule is short and no row missing, so what changes from step to step is uniform
    const uint32_t at_a = ((uint32_t)row * (uint32_t)A.K + g * 8) * (uint32_t)sizeof(T);
    auto fetch_whole = [&](int k0) {
        int row_ = row;
        asm volatile("" : "+v"(row_));
        auto at_b = [&](int i) {
            return (__umul24(row_ + i * RP < left_b ? row_ + i * RP : left_b, A.ldb) + g * 8) * (CUT ? 2u : (uint32_t)sizeof(T));
        };
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const long long to = (long long)(i * RP) * A.K + k0;
            ga[i] = ld_gran<T>(ba + to, at_a);
            if (!FWD && sloped) gs[i] = ld_slope<T>(bs + to, at_a / (uint32_t)sizeof(T) * (uint32_t)sizeof(ST));
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if constexpr (CUT) {
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    gc[i][p] = *reinterpret_cast<const u32x4 *>(bb + p * plane + (long long)k0 * 2 + at_b(i));
            } else {
                gb[i] = ld_gran<T>(bb + (long long)k0 * (int)sizeof(T), at_b(i));
            }
        }
    };
    auto fetch = [&](int k0) {
        if constexpr (WHOLE) return fetch_whole(k0);
        const int k = k0 + g * 8, ka = SHORT ? k : (k < A.K - 8 ? k : A.K - 8), kb = SHORT && !CUT ? k : (k < last ? k : last);
        // Rows' offsets in elements, made again at every step: kept, they are the registers that do not fit and
        // went to scratch memory.  The compiler must not know that they are the same each time.
        int row_ = row;
        asm volatile("" : "+v"(row_));
        auto row_a = [&](int i) { return __umul24(row_ + i * RP < left_a ? row_ + i * RP : left_a, A.K); };
        auto row_b = [&](int i) { return __umul24(row_ + i * RP < left_b ? row_ + i * RP : left_b, A.ldb); };
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            if constexpr (SHORT) {
                ga[i] = ld_gran_short<T>(ba, (row_a(i) + ka) * (uint32_t)sizeof(T), A.K - k);
                if (!FWD && sloped) gs[i] = ld_slope_short<T>(bs, (row_a(i) + ka) * (uint32_t)sizeof(ST), A.K - k);
            } else {
                ga[i] = ld_gran<T>(ba, (row_a(i) + ka) * (uint32_t)sizeof(T));
                if (!FWD && sloped) gs[i] = ld_slope<T>(bs, (row_a(i) + ka) * (uint32_t)sizeof(ST));
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if constexpr (CUT) {
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    gc[i][p] = *reinterpret_cast<const u32x4 *>(bb + p * plane + (row_b(i) + kb) * 2u);
            } else if constexpr (SHORT) {
                gb[i] = ld_gran_short<T>(bb, (row_b(i) + kb) * (uint32_t)sizeof(T), A.K - k);
            } else {
                gb[i] = ld_gran<T>(bb, (row_b(i) + kb) * (uint32_t)sizeof(T));
            }
        }
    };
    f32x16v acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
    bool twice = false;
    if constexpr (TWO) {        // (in front of the first loads, which take as long)
        const int groups = (A.N - n0 < BN ? A.N - n0 + 31 : BN) / 32;
        const uint8_t *bad = A.bad + (long long)(n0 / 32) * A.bad_cols;
        uint32_t any = 0;
        for (int i = threadIdx.x; i < groups * A.bad_cols; i += THREADS) any |= bad[i];
        fetch(k_first);
        twice = __builtin_amdgcn_readfirstlane(__syncthreads_or(any)) != 0;
    } else {
        fetch(k_first);
    }
    for (int k0 = k_first; k0 < k_end; k0 += TA::BK) {
        // the row's last, partial step: what a granule holds of the one before it is dropped.  An image has
        // zeros behind K instead of a step back, in its place: A must line up, so it is moved down there.
        const bool end = !SHORT && !WHOLE && k0 + TA::BK > A.K;
        const int k = k0 + g * 8, over = k > A.K - 8 ? k - (A.K - 8) : 0;
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            if constexpr (TWO) {
                if (end) drop(ga[i], over);
                TA::put2(la, row + i * RP, g, with_slope<T>(ga[i], gs[i], A.slope_scale), twice);
                continue;
            } else {
                if (!FWD && sloped) ga[i] = to_gran<T>(with_slope<T>(ga[i], gs[i], A.slope_scale));
                if (end) {
                    if constexpr (CUT) shift_down<T>(ga[i].w, over);
                    else drop(ga[i], over);
                }
                TA::put(la, row + i * RP, g, ga[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (BN < RP && row >= BN) continue;
            if constexpr (CUT) {
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<u32x4 *>(lb + p * TB::PLANE + TB::at(row + i * RP, g)) = gc[i][p];
            } else {
                if (end) drop(gb[i], over);
                TB::put(lb, row + i * RP, g, gb[i]);
            }
        }
        __syncthreads();
        if (k0 + TA::BK < k_end) fetch(k0 + TA::BK);
        tile_mma<T, TA, TB, MI, NI>(la, lb, wm, wn, lane, acc);
        __syncthreads();
    }
    if (TWO && twice)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[i][j][q] *= 0.5f;
    if constexpr (PART) {
        float *part = A.part + split * A.M * A.N;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const long long m = m0 + wm + i * 32 + acc_row(q, lane >> 5);
                    const int n = n0 + wn + j * 32 + (lane & 31);
                    if (m < A.M && n < A.N) part[m * A.N + n] = acc[i][j][q];
                }
        return;
    }
    // epilogue: a wave turns its blocks 16 rows at a time through LDS of its own into row pieces of 8
    float *le = reinterpret_cast<float *>(smem) + wave * 16 * LD;
    constexpr int PR = NI * 4, RI = 64 / PR;        // pieces a row, rows at once
    const int half = lane >> 5, c8 = (lane % PR) * 8, rr = lane / PR;
    const int n = n0 + wn + c8;
    const int have = A.N - n;                       // columns of this piece that exist
    // the residual's pieces are on their way before they are used: of a 32-row block for f32, of 16 rows for
    // 16-bit types, whose four waves a SIMD have no registers for more
    constexpr int PP = 16 / RI, AHEAD = IsF32<T>::value ? 2 : 1;
    Gran<T> res[AHEAD][PP];
    auto fetch_res = [&](int i, int h0) {
        const T *br = static_cast<const T *>(A.res) + (m0 + wm) * A.N;
        const long long left = A.M - 1 - (m0 + wm);
        const int nc = SHORT_N || n <= A.N - 8 ? n : A.N - 8;
#pragma unroll
        for (int h = 0; h < AHEAD; ++h)
#pragma unroll
            for (int p = 0; p < PP; ++p) {
                const int r = i * 32 + (h0 + h) * 16 + p * RI + rr;
                // a wave whose rows all lie behind the matrix reads the row before them
                const long long at = (r < left ? r : left) * (long long)A.N + nc;
                if constexpr (SHORT_N) res[h][p] = ld_gran_short<T>(br + at, 0, have);
                else res[h][p] = ld_gran<T>(br + at, 0);
            }
    };
    Gran<T> bias;       // (as it lies in memory: half the registers of f32 ones for 16-bit types)
    if (FWD) bias = ld_gran_short<T>(A.bias, (uint32_t)n * sizeof(T), A.bias ? have : 0);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (FWD && A.res && h % AHEAD == 0) fetch_res(i, h);
            // the wave's own LDS, in order: what it stored before is read before it stores again
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int q = 0; q < 8; ++q) le[acc_row(q, half) * LD + j * 32 + (lane & 31)] = acc[i][j][h * 8 + q];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int p = 0; p < 16 / RI; ++p) {
                const long long m = m0 + wm + i * 32 + h * 16 + p * RI + rr;
                if (m >= A.M || m < m_first || have <= 0) continue;      // (before m_first: another tile's)
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = le[(p * RI + rr) * LD + c8 + k];
                if constexpr (IsF32<T>::value) {        // see the head of this file
                    bool fine = true;
#pragma unroll
                    for (int k = 0; k < 8; ++k) fine = fine && fabsf(v[k]) < INFINITY;
                    if (!fine) {
                        float *row = le + (p * RI + rr) * LD + c8;      // this lane's own eight
#pragma unroll 1
                        for (int k = 0; k < 8; ++k)
                            if (k < have && !(fabsf(row[k]) < INFINITY)) row[k] = plain_dot<FWD>(A, m, n + k);
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = row[k];
                    }
                }
                if (FWD && !SHORT_N && have < 8 && A.res) shift_down<T>(res[h % AHEAD][p].w, 8 - have);
                epi_piece<T, FWD>(A, m, n, have, v, bias, res[h % AHEAD][p]);
            }
        }
    }
}

// The sums of a split contraction, joined in order, and what the product's own epilogue would have done
template <class T, bool FWD> __global__ __launch_bounds__(256) void lin_join_kernel(const LinArgs A) {
    const long long at = blockIdx.x * 256ll + threadIdx.x, size = A.M * A.N;
    if (at >= size) return;
    float v = 0.f;
#pragma unroll 8
    for (int q = 0; q < A.splits; ++q) v += A.part[q * size + at];
    const long long m = at / A.N;
    const int n = (int)(at - m * A.N);
    if (IsF32<T>::value && !(fabsf(v) < INFINITY)) v = plain_dot<FWD>(A, m, n);
    if constexpr (FWD) {
        const float z = v + (A.bias ? (float)static_cast<const T *>(A.bias)[n] : 0.f);
        GATMI_WITH_ACT(A.act, {
            float d;
            v = act_both<ACT, IsF32<T>::value>(z, d);
            if (A.slope) static_cast<typename SlopeOf<T>::type *>(A.slope)[at] = slope_out<T, ACT>(d);
        });
        if (A.res) v += (float)static_cast<const T *>(A.res)[at];
    }
    static_cast<T *>(A.C)[at] = (T)v;
}

// A tile of the transposed product in LDS, as it lies in memory: contraction steps (rows of the matrix) by
// C channels, PIECES planes.  Fragments are read with the transposing LDS load: 16 lanes fetch a block of
// 4 steps x 16 channels, four channels each, and every lane comes back with one channel's four steps.  The
// 64-byte pieces of a row change places by the row's last two bits, so that the four rows of a block lie in
// different banks.  (Rows padded by 64 bytes do the same, but then two blocks of f32 tiles miss fitting a CU.)
template <class T, int C, int PIECES = Mul<T>::PIECES> struct TileT {
    static constexpr int BK = Mul<T>::BK, P = PIECES;
    static constexpr int STRIDE = C * 2, PLANE = BK * STRIDE, BYTES = PLANE * P;
    static __device__ __forceinline__ int at(int row, int col) { return row * STRIDE + ((col * 2) ^ ((row & 3) << 6)); }
    static __device__ __forceinline__ void put(char *lds, int row, int col, const Gran<T> &v) {
        char *to = lds + at(row, col);
        if constexpr (P == 1) {
            *reinterpret_cast<u32x4 *>(to) = u32x4{v.w[0], v.w[1], v.w[2], v.w[3]};
        } else {
            uint32_t q[3][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                cut3(__uint_as_float(v.w[2 * i]), __uint_as_float(v.w[2 * i + 1]), q[0][i], q[1][i], q[2][i]);
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<u32x4 *>(to + p * PLANE) = u32x4{q[p][0], q[p][1], q[p][2], q[p][3]};
        }
    }
    static __device__ __forceinline__ void put2(char *lds, int row, int col, const VecF<8> &v, bool twice) {
        static_assert(P == 2, "a tile of halves");
        Gran<T> q[2];
        split2<T>(v, q[0], q[1], twice);
#pragma unroll
        for (int p = 0; p < 2; ++p)
            *reinterpret_cast<u32x4 *>(lds + p * PLANE + at(row, col)) = u32x4{q[p].w[0], q[p].w[1], q[p].w[2], q[p].w[3]};
    }
    // channels col0 .. col0 + 31, steps 16 s + 8 half .. + 7 of this lane's channel
    static __device__ __forceinline__ u32x4 frag(const char *lds, int p, int s, int col0, int lane) {
        typedef short v4s __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) v4s *lds_ptr;
        const int row = 16 * s + (lane >> 5) * 8 + ((lane & 15) >> 2), col = col0 + (lane & 16) + (lane & 3) * 4;
        const char *from = lds + p * PLANE + at(row, col);
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(from));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(from + 4 * STRIDE));
        return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// Whether this block's sums have to be taken again, where dz is two numbers: some sum is not finite, and so is some
// factor of the other side among `rows` rows (`stride` apart) of `cols` columns, which met a lo of 0 or of the other
// sign than hi.  (An infinity of dz alone comes out right.)  They are, by a second pass with hi for lo: twice the sum
// of the rounded dz, whose infinities and NaN are those of the formula; what was finite stays as it is.
template <class T>
__device__ __forceinline__ bool redo(const f32x16v (&acc)[2][2], const T *b, long long rows, long long stride, int cols) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) s = fmaf(acc[i][j][q], 0.f, s);       // NaN once one is not finite
    if (!__syncthreads_or(s != 0.f)) return false;
    // as many rows at once as fit the block side by side
    const int threads = blockDim.x, wide = cols < threads ? cols : threads, high = threads / wide;
    const int c0 = threadIdx.x % wide, r0 = threadIdx.x / wide;
    bool bad = false;
    if (r0 < high)
        for (int c = c0; c < cols; c += wide)
#pragma unroll 8
            for (long long r = r0; r < rows; r += high) bad |= !(fabsf((float)b[r * stride + c]) < INFINITY);
    return __syncthreads_or(bad);
}

// The wide form is 512 threads and one block a CU (its registers), so nothing but its own loads in flight hides
// the memory: two steps' for 16-bit types, 0.82 -> 0.71 ms for [2449029, 256] x [2449029, 256] bf16 together with
// the XCD's order.  f32 gains nothing from it: 104 us for [100000, 240] x [100000, 240] either way.
//
// dW slabs: part[split][n][k] = sum over the split's rows of dz[m][n] x[m][k], dz = A (* aslope) [M, N],
// x = B [M, K]; the blocks of the first column of tiles also leave dz's column sums.  SHORT: N or K < 8.
template <class T, int BN, bool SHORT, bool TWO> __global__ __launch_bounds__(2 * BN) void lin_tn_kernel(const LinArgs A) {
    static_assert(!TWO || !IsF32<T>::value, "dz of 16-bit tensors");
    typedef TileT<T, kBM, TWO ? 2 : Mul<T>::PIECES> TA;
    typedef TileT<T, BN> TB;
    constexpr int THREADS = 2 * BN, WN = BN / 64, GA = kBM / 8, GB = BN / 8;
    constexpr int RA = THREADS / GA, RB = THREADS / GB, NA = TA::BK / RA, NB = TA::BK / RB;
    __shared__ __attribute__((aligned(16))) char smem[TA::BYTES + TB::BYTES];
    static_assert(TA::BYTES + TB::BYTES >= RA * kBM * 4, "the column sums fit");
    char *la = smem, *lb = smem + TA::BYTES;
    // the tiles of a split read the same rows: each XCD (block index mod 8) has a contiguous range of
    // (split, tile), so that they meet in its L2
    const long long item = (long long)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (item >= A.tiles * A.splits) return;
    const long long split = item / A.tiles;
    const int tile = (int)(item - split * A.tiles);
    const int n0 = tile / (int)A.tiles_n * kBM, k0 = tile % (int)A.tiles_n * BN;
    const long long r0 = split * A.per_split, r1 = r0 + A.per_split < A.M ? r0 + A.per_split : A.M;
    const T *pa = static_cast<const T *>(A.A), *pb = static_cast<const T *>(A.B);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave / WN) * 64, wn = (wave % WN) * 64;
    typedef typename SlopeOf<T>::type ST;
    const bool sloped = TWO || A.aslope, sums = (A.dbpart || A.db) && k0 == 0;
    // Two steps' pieces where the registers are there: while one is stored, the other is on its way.
    constexpr int SETS = !IsF32<T>::value && BN == 256 ? 2 : 1;
    Gran<T> ga_[SETS][NA], gb_[SETS][NB];
    SlopeGran<T> gs_[SETS][NA];
    VecF<8> db;
#pragma unroll
    for (int k = 0; k < 8; ++k) db.e[k] = 0.f;
    // a thread's pieces: eight channels, rows ta + i * RA (tb + i * RB).  A piece that would run over the last
    // channel is loaded from the last eight and moved to its place.
    const int ta = threadIdx.x / GA, ja = threadIdx.x % GA * 8, tb = threadIdx.x / GB, jb = threadIdx.x % GB * 8;
    const bool edge_a = !SHORT && n0 + kBM > A.N, edge_b = !SHORT && k0 + BN > A.K;
    int ca = n0 + ja, cb = k0 + jb, over_a = 0, over_b = 0;
    if (!SHORT && ca > A.N - 8) {
        over_a = ca - (A.N - 8);
        ca = A.N - 8;
    }
    if (!SHORT && cb > A.K - 8) {
        over_b = cb - (A.K - 8);
        cb = A.K - 8;
    }
    auto fetch = [&](auto set, long long r) {
        Gran<T>(&ga)[NA] = ga_[decltype(set)::value], (&gb)[NB] = gb_[decltype(set)::value];
        SlopeGran<T>(&gs)[NA] = gs_[decltype(set)::value];
        if (r > r1 - 1) r = r1 - 1;          // behind the end: loaded all the same, never used
        const T *ra = pa + r * A.N, *rb = pb + r * A.K;
        const ST *rs = static_cast<const ST *>(A.aslope) + r * A.N;
        const int left = (int)(r1 - 1 - r < TA::BK ? r1 - 1 - r : TA::BK);      // rows behind the last repeat it
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const uint32_t m = ta + i * RA < left ? ta + i * RA : left, at = m * (uint32_t)A.N + ca;
            if constexpr (SHORT) {
                ga[i] = ld_gran_short<T>(ra, at * (uint32_t)sizeof(T), A.N - ca);
                if (sloped) gs[i] = ld_slope_short<T>(rs, at * (uint32_t)sizeof(ST), A.N - ca);
            } else {
                ga[i] = ld_gran<T>(ra, at * (uint32_t)sizeof(T));
                if (sloped) gs[i] = ld_slope<T>(rs, at * (uint32_t)sizeof(ST));
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint32_t m = tb + i * RB < left ? tb + i * RB : left, at = m * (uint32_t)A.K + cb;
            if constexpr (SHORT) gb[i] = ld_gran_short<T>(rb, at * (uint32_t)sizeof(T), A.K - cb);
            else gb[i] = ld_gran<T>(rb, at * (uint32_t)sizeof(T));
        }
    };
    f32x16v acc[2][2];
    auto step = [&](auto set, long long r, bool twice) __attribute__((always_inline)) {
        Gran<T>(&ga)[NA] = ga_[decltype(set)::value], (&gb)[NB] = gb_[decltype(set)::value];
        SlopeGran<T>(&gs)[NA] = gs_[decltype(set)::value];
        const bool end = r + TA::BK > r1;
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            if (edge_a) {
                shift_down<T>(ga[i].w, over_a);
                if (sloped) shift_down<T>(gs[i].w, over_a);
            }
            if (end && r + ta + i * RA >= r1) {        // no such row: zeros, slope and all
                shift_down<T>(ga[i].w, 8);
                if (sloped) shift_down<T>(gs[i].w, 8);
            }
            if (sloped) {
                const VecF<8> v = with_slope<T>(ga[i], gs[i], A.slope_scale);
                if (sums && !twice)
#pragma unroll
                    for (int k = 0; k < 8; ++k) db.e[k] += v.e[k];     // before the rounding
                if constexpr (TWO) {
                    TA::put2(la, ta + i * RA, ja, v, twice);
                    continue;
                }
                ga[i] = to_gran<T>(v);
            } else if (sums) {
                const VecF<8> v = gran_values<T>(ga[i]);
#pragma unroll
                for (int k = 0; k < 8; ++k) db.e[k] += v.e[k];
            }
            if constexpr (!TWO) TA::put(la, ta + i * RA, ja, ga[i]);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if (edge_b) shift_down<T>(gb[i].w, over_b);
            if (end && r + tb + i * RB >= r1) shift_down<T>(gb[i].w, 8);
            TB::put(lb, tb + i * RB, jb, gb[i]);
        }
        __syncthreads();
        fetch(set, r + SETS * TA::BK);
#pragma unroll
        for (int s = 0; s < TA::BK / 16; ++s) {
            u32x4 a[2][TA::P], b[2][TB::P];
#pragma unroll
            for (int p = 0; p < TA::P; ++p)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    a[i][p] = TA::frag(la, p, s, wm + i * 32, lane);
                    if (p < TB::P) b[i][p < TB::P ? p : 0] = TB::frag(lb, p, s, wn + i * 32, lane);
                }
            mma_pieces<T, TA::P, 2, 2>(a, b, acc);
        }
        __syncthreads();
    };
    auto sweep = [&](bool twice) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
        if (r0 >= r1) return;
        typedef std::integral_constant<int, 0> First;
        typedef std::integral_constant<int, SETS - 1> Second;
        fetch(First{}, r0);
        if constexpr (SETS == 2) fetch(Second{}, r0 + TA::BK);
        for (long long r = r0; r < r1; r += SETS * TA::BK) {
            step(First{}, r, twice);
            if constexpr (SETS == 2)
                if (r + TA::BK < r1) step(Second{}, r + TA::BK, twice);
        }
    };
    sweep(false);
    if (sums) {      // [RA][128] partial sums, added in order
        float *red = reinterpret_cast<float *>(smem);
#pragma unroll
        for (int k = 0; k < 8; ++k) red[ta * kBM + ja + k] = db.e[k];
        __syncthreads();
        if (threadIdx.x < kBM && n0 + (int)threadIdx.x < A.N) {
            float s = 0.f;
            for (int q = 0; q < RA; ++q) s += red[q * kBM + threadIdx.x];
            if (A.db) static_cast<T *>(A.db)[n0 + threadIdx.x] = (T)s;
            else A.dbpart[split * A.N + n0 + threadIdx.x] = s;
        }
    }
    if (!A.part && !A.dw) return;       // the bias alone
    float *part = A.part + split * (long long)A.N * A.K;
    // f(element's place in dW, its sum)
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const int n = n0 + wm + i * 32 + acc_row(q, lane >> 5), k = k0 + wn + j * 32 + (lane & 31);
                    if (n < A.N && k < A.K) f(n, k, acc[i][j][q]);
                }
    };
    each([&](int n, int k, float v) {
        if (IsF32<T>::value && !(fabsf(v) < INFINITY)) {
            v = 0.f;
            for (long long m = r0; m < r1; ++m) {
                float d = (float)pa[m * A.N + n];
                if (sloped) d *= static_cast<const float *>(A.aslope)[m * A.N + n];
                v = fmaf(d, (float)pb[m * A.K + k], v);
            }
        }
        if (A.dw) static_cast<T *>(A.dw)[(long long)n * A.K + k] = (T)v;
        else part[(long long)n * A.K + k] = v;
    });
    if constexpr (TWO)
        if (redo<T>(acc, pb + r0 * A.K + k0, r1 - r0, A.K, A.K - k0 < BN ? A.K - k0 : BN)) {
            sweep(true);
            each([&](int n, int k, float v) {
                const long long at = (long long)n * A.K + k;
                if (A.dw) {
                    T *o = static_cast<T *>(A.dw) + at;
                    if (!(fabsf((float)*o) < INFINITY)) *o = (T)v;
                } else if (!(fabsf(part[at]) < INFINITY)) {
                    part[at] = v;
                }
            });
        }
}

// A few rows (serving): one wave a column of y, lanes along the contraction, f32 multiply-adds whatever the
// type.  The weights are read once, by as many waves as there are columns.
template <class T, int MR> __global__ __launch_bounds__(256) void lin_rows_kernel(const LinArgs A) {
    constexpr int V = 16 / sizeof(T);
    const int lane = threadIdx.x & 63;
    const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= A.N) return;
    const T *w = static_cast<const T *>(A.B) + (long long)n * A.K, *x = static_cast<const T *>(A.A);
    const int M = (int)A.M;
    float acc[MR];
#pragma unroll
    for (int r = 0; r < MR; ++r) acc[r] = 0.f;
    const int whole = A.K / V * V;
#pragma unroll 2
    for (int k = lane * V; k < whole; k += 64 * V) {
        const VecF<V> wv = ldv<T, V>(w + k);
#pragma unroll
        for (int r = 0; r < MR; ++r) {
            const VecF<V> xv = ldv<T, V>(x + (long long)(r < M ? r : M - 1) * A.K + k);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[r] = fmaf(xv.e[i], wv.e[i], acc[r]);
        }
    }
    if (whole + lane < A.K) {
        const float wl = (float)w[whole + lane];
#pragma unroll
        for (int r = 0; r < MR; ++r) acc[r] = fmaf((float)x[(long long)(r < M ? r : M - 1) * A.K + whole + lane], wl, acc[r]);
    }
    float z = 0.f;
#pragma unroll
    for (int r = 0; r < MR; ++r) {
        const float s = head_sum<64>(acc[r], 64);
        if (lane == r) z = s;      // lane r ends with row r
    }
    if (lane >= M) return;
    const long long at = (long long)lane * A.N + n;
    z += A.bias ? (float)static_cast<const T *>(A.bias)[n] : 0.f;
    float y = z;
    GATMI_WITH_ACT(A.act, {
        float d;
        y = act_both<ACT, IsF32<T>::value>(z, d);
        if (A.slope) static_cast<typename SlopeOf<T>::type *>(A.slope)[at] = slope_out<T, ACT>(d);
    });
    if (A.res) y += (float)static_cast<const T *>(A.res)[at];
    static_cast<T *>(A.C)[at] = (T)y;
}

// dW = sum of the slabs and db = sum of the splits' column sums, in order: the first `dw_blocks` blocks and the
// others.  64 values by 4 groups of slabs a block (8 by 32 for db): few values and hundreds of slabs still make
// many loads
template <class T> __global__ __launch_bounds__(256) void lin_slabs_kernel(const float *part, int splits, long long size, T *dw,
                                                                          int dw_blocks, const float *dbpart, int N, T *db) {
    __shared__ double red[256];
    if ((int)blockIdx.x < dw_blocks) {
        const int lane = threadIdx.x & 63, grp = threadIdx.x >> 6;
        const long long i = blockIdx.x * 64ll + lane;
        float s = 0.f;
        if (i < size)
#pragma unroll 8
            for (int q = grp; q < splits; q += 4) s += part[q * size + i];
        red[threadIdx.x] = s;
        __syncthreads();
        if (grp == 0 && i < size) dw[i] = (T)(float)(((s + red[64 + lane]) + red[128 + lane]) + red[192 + lane]);
        return;
    }
    const int c = (blockIdx.x - dw_blocks) * 8 + (threadIdx.x & 7), rg = threadIdx.x >> 3;
    double s = 0.0;
    if (c < N)
#pragma unroll 4
        for (int b = rg; b < splits; b += 32) s += dbpart[(long long)b * N + c];
    red[threadIdx.x] = s;
    __syncthreads();
    if (rg == 0 && c < N) {
        for (int q = 1; q < 32; ++q) s += red[threadIdx.x + q * 8];
        db[c] = (T)(float)s;
    }
}

// The weights as the products take them: rows of `ld` (a multiple of 8, zeros behind the end), the matrix
// itself (TR: transposed, out[k][n] = w[n][k]), f32 as three planes of bf16 pieces.  bad (or null): a byte a block,
// whether its 32 x 32 hold an infinity or NaN.
template <class T, bool TR> __global__ __launch_bounds__(256) void lin_image_kernel(const T *w, int N, int K, int ld, void *out,
                                                                                        uint8_t *bad) {
    __shared__ T t[32][33];
    const int R = TR ? K : N, S = TR ? N : K;       // rows and columns of the image
    const int s0 = blockIdx.x * 32, r0 = blockIdx.y * 32, x = threadIdx.x & 31, y = threadIdx.x >> 5;
    int odd = 0;
    for (int i = y; i < 32; i += 8) {
        const int n = TR ? s0 + i : r0 + i, k = TR ? r0 + x : s0 + x;
        const T v = n < N && k < K ? w[(long long)n * K + k] : (T)0.f;
        t[TR ? x : i][TR ? i : x] = v;
        if (!(fabsf((float)v) < INFINITY)) odd = 1;
    }
    const int any = __syncthreads_or(odd);
    if (bad && threadIdx.x == 0) bad[(long long)blockIdx.y * gridDim.x + blockIdx.x] = (uint8_t)(any != 0);
    for (int i = y; i < 32; i += 8) {
        if (r0 + i >= R || s0 + x >= ld) continue;
        const long long at = (long long)(r0 + i) * ld + s0 + x;
        if constexpr (IsF32<T>::value) {
            uint32_t p0, p1, p2;
            cut3(t[i][x], 0.f, p0, p1, p2);
            uint16_t *o = static_cast<uint16_t *>(out);
            const long long plane = (long long)R * ld;
            o[at] = (uint16_t)p0;
            o[plane + at] = (uint16_t)p1;
            o[2 * plane + at] = (uint16_t)p2;
        } else {
            static_cast<T *>(out)[at] = t[i][x];
        }
    }
    (void)S;
}

static int lin_check(const gatmi_linear *l) {
    GATMI_REQUIRE(l, "null linear descriptor");
    GATMI_REQUIRE(l->dtype >= GATMI_F32 && l->dtype <= GATMI_F16, "linear: unknown element type %d", l->dtype);
    GATMI_REQUIRE(l->act >= GATMI_ACT_NONE && l->act <= GATMI_ACT_GELU, "linear: unknown activation %d", l->act);
    GATMI_REQUIRE(l->in_features >= 1 && l->in_features <= 65536 && l->out_features >= 1 && l->out_features <= 65536,
                  "linear: %d -> %d features out of range (1 .. 65536)", l->in_features, l->out_features);
    GATMI_REQUIRE(l->rows >= 0 && l->rows < (1ll << 31), "linear: %lld rows out of range", (long long)l->rows);
    return GATMI_OK;
}

// From this many rows on the f32 forward reads its weights as pieces cut once, not by every block
constexpr long long kCutRows = 2048;
// Up to this many rows go without the matrix cores, but 16-bit ones above four where the contraction is split:
// 16 rows of [1024, 1024] bf16 take 8.0 us so and 5.9 in pieces, f32 5.5 and 7.3
constexpr int kFewRows = 16;

// Few tiles and a long contraction: a step of it takes a lone block 0.5 us (f32: 0.7), most of that waiting on
// itself, and the chip is empty beside it.  Pieces of at least two steps, as many as give two blocks a CU, and a
// kernel that joins them (2 us): from six (f32) or eight steps saved on, while the tiles are at most half the CUs.
// [64, 1024] x [1024, 1024] bf16 12.0 -> 6.8 us, f32 29.7 -> 8.8; [1024, 1024] x [1024, 1024], 256 tiles, bf16
// 12.8 -> 16.3, so not there.
struct LinSplitK {
    int splits, k_split;
    size_t bytes;
};
static LinSplitK lin_split_k(long long M, int N, int K, int dtype) {
    LinSplitK S = {1, K, 0};
    if (M < 1) return S;
    const int bk = dtype == GATMI_F32 ? 32 : 64, steps = (K + bk - 1) / bk;
    const long long tiles = (M + 63) / 64 * ((N + 63) / 64), room = 2ll * device_cus() / tiles;
    const long long want = room < (steps + 1) / 2 ? room : (steps + 1) / 2;
    if (want < 2 || room < 4) return S;
    const int each = (int)((steps + want - 1) / want);
    if (steps - each < (dtype == GATMI_F32 ? 6 : 8)) return S;
    S.k_split = each * bk;
    S.splits = (steps + each - 1) / each;
    S.bytes = align_up((size_t)S.splits * M * N * 4);
    return S;
}

struct LinGeom {
    int splits;
    bool wide;                      // dW's tiles: 256 columns of x, for which dz is made once, instead of 128
    long long per_split;
    int ldf, ldb;                   // row lengths of the weight images, forward and transposed
    size_t image_f, image_b, slabs, dbpart;     // bytes; slabs and dbpart are used by more than one split only
    size_t bad_b;                   // of image_b, behind the image: a byte for every 32 x 32 (dz as two numbers)
    LinSplitK fwd, dx;
    bool image_fwd;                 // the forward takes an image
    bool few;                       // ... or the few-row kernel
};

static long long lin_dw_tiles(const gatmi_linear *l, bool wide) {
    const int bn = wide ? 256 : 128;
    return ((l->out_features + kBM - 1ll) / kBM) * ((l->in_features + bn - 1ll) / bn);
}
// dz as two numbers: where it does not fit the tensors' type
static bool lin_two(const gatmi_linear *l) {
    return l->dtype != GATMI_F32 && l->act != GATMI_ACT_NONE && l->act != GATMI_ACT_RELU;
}

static LinGeom lin_geom(const gatmi_linear *l) {
    LinGeom G;
    memset(&G, 0, sizeof(G));
    const size_t el = l->dtype == GATMI_F32 ? 6 : 2;
    G.wide = l->in_features > 128;
    const long long tiles = lin_dw_tiles(l, G.wide);
    // The rows are split so that the blocks fill the chip a whole number of times: a wide block's registers
    // leave room for no second one on its CU, of narrow ones two fit.  In units of a row of one block: a round
    // of blocks takes its rows and about 256 more for its start and its slab, a slab's way through memory
    // N K / 2^14.  At least 256 rows a split.
    const long long slots = device_cus() * (G.wide ? 1ll : 2ll), most = (l->rows + 255) / 256;
    long long s = 1, best = -1;
    for (long long rounds = 1; rounds <= 4; ++rounds) {
        long long c = rounds * slots / tiles;
        c = c < 1 ? 1 : (c > most && most > 0 ? most : c);
        const long long t = (c * tiles + slots - 1) / slots * (l->rows / c + 256) +
                            c * ((long long)l->out_features * l->in_features >> 14);
        if (best < 0 || t < best) {
            best = t;
            s = c;
        }
    }
    const int bk = l->dtype == GATMI_F32 ? 32 : 64;
    G.per_split = ((l->rows + s - 1) / s + bk - 1) / bk * bk;
    if (G.per_split < bk) G.per_split = bk;
    G.splits = (int)((l->rows + G.per_split - 1) / G.per_split);
    if (G.splits < 1) G.splits = 1;
    G.ldf = (l->in_features + 7) / 8 * 8;
    G.ldb = (l->out_features + 7) / 8 * 8;
    G.image_fwd = l->dtype == GATMI_F32 && l->rows >= kCutRows;
    G.fwd = lin_split_k(l->rows, l->out_features, l->in_features, l->dtype);
    G.few = l->rows <= 4 || (l->rows <= kFewRows && (l->dtype == GATMI_F32 || G.fwd.splits == 1));
    if (G.few) G.fwd = {1, l->in_features, 0};
    G.dx = lin_split_k(l->rows, l->in_features, l->out_features, l->dtype);
    G.image_f = G.image_fwd ? align_up((size_t)l->out_features * G.ldf * el) : 0;
    G.bad_b = lin_two(l) ? align_up((size_t)((l->in_features + 31) / 32) * ((G.ldb + 31) / 32)) : 0;
    G.image_b = align_up((size_t)l->in_features * G.ldb * el) + G.bad_b;
    G.slabs = align_up((size_t)G.splits * l->in_features * l->out_features * 4);
    G.dbpart = align_up((size_t)G.splits * l->out_features * 4);
    return G;
}

template <class T, bool TWO, int BM, int BN, int WM, int WN, bool FWD, bool CUT, bool SHORT = false, bool SHORT_N = false,
          bool WHOLE = false>
static void lin_go(LinArgs &A, hipStream_t st) {
    typedef typename SlopeOf<T>::type ST;
    A.tiles_n = (A.N + BN - 1) / BN;
    // a launch counts its threads in 32 bits: 2^23 blocks of 256 at most.  (The rows before a later slice are
    // there to be read, so its last tile may start in them.)
    const long long rows = A.M, most = (1ll << 23) / A.tiles_n * BM;
    auto move = [](auto *p, long long bytes) { return p ? reinterpret_cast<decltype(p)>((uintptr_t)p + bytes) : p; };
    for (long long m = 0; m < rows; m += most) {
        LinArgs S = A;
        S.M = rows - m < most ? rows - m : most;
        S.A = move(A.A, m * A.K * sizeof(T));
        S.aslope = move(A.aslope, m * A.K * sizeof(ST));
        S.res = move(A.res, m * A.N * sizeof(T));
        S.C = move(A.C, m * A.N * sizeof(T));
        S.slope = move(A.slope, m * A.N * sizeof(ST));
        S.tiles = (S.M + BM - 1) / BM * S.tiles_n;
        const unsigned grid = (unsigned)((S.tiles + 7) / 8 * 8);
        hipLaunchKernelGGL((lin_nt_kernel<T, BM, BN, WM, WN, FWD, CUT, SHORT, SHORT_N, false, WHOLE, TWO>), dim3(grid), dim3(WM * WN * 64), 0,
                           st, S);
    }
}
// The tile.  While 128 x 128 ones would be fewer than two a CU, 64 x 64: a lone block of the large ones waits
// for itself ([4096, 64] x [64, 1024] f32 24.7 -> 16.7 us, bf16 11.1 -> 8.1; with 3 a CU [8192, 1024] x
// [1024, 1024] f32 loses, 117 -> 134).  Narrow results take narrow tiles, 128 x 32 from one a CU on.  Where dz is two
// numbers a 128 x 128 tile's 48 KB of LDS and 184 registers leave two blocks a CU; half the rows leave three or four, and
// up to 256 columns a tile make dz once: dx of [2449029, 256] x [256, 256] bf16 1.36 -> 1.02 ms, to 128 columns 0.77 -> 0.69.
template <class T, bool FWD, bool CUT, bool TWO> static void lin_launch_nt(LinArgs A, const LinSplitK &S, hipStream_t st) {
    if (S.splits > 1) {
        A.splits = S.splits;
        A.k_split = S.k_split;
        A.tiles_n = (A.N + 63) / 64;
        A.tiles = (A.M + 63) / 64 * A.tiles_n;
        const unsigned grid = (unsigned)((A.tiles * A.splits + 7) / 8 * 8);
        hipLaunchKernelGGL((lin_nt_kernel<T, 64, 64, 2, 2, FWD, CUT, false, false, true, false, TWO>), dim3(grid), dim3(256), 0, st, A);
        hipLaunchKernelGGL((lin_join_kernel<T, FWD>), dim3((unsigned)((A.M * A.N + 255) / 256)), dim3(256), 0, st, A);
        return;
    }
    const long long big = (A.M + 127) / 128 * ((A.N + 127) / 128);
    if (A.K < 8) lin_go<T, TWO, 64, 64, 2, 2, FWD, CUT, true, true>(A, st);
    else if (A.N < 8) lin_go<T, TWO, 128, 32, 4, 1, FWD, CUT, false, true>(A, st);
    else if (A.N <= 32 && big >= device_cus()) lin_go<T, TWO, 128, 32, 4, 1, FWD, CUT>(A, st);
    else if (big < 2 * device_cus()) lin_go<T, TWO, 64, 64, 2, 2, FWD, CUT>(A, st);
    else if (A.N <= 64) lin_go<T, TWO, 128, 64, 4, 1, FWD, CUT>(A, st);
    else {
        const bool whole = !IsF32<T>::value && A.K % Mul<T>::BK == 0 && A.M >= 128;
        if constexpr (TWO) {
            if (A.N <= 128) whole ? lin_go<T, TWO, 64, 128, 2, 2, FWD, CUT, false, false, true>(A, st) : lin_go<T, TWO, 64, 128, 2, 2, FWD, CUT>(A, st);
            else whole ? lin_go<T, TWO, 64, 256, 1, 4, FWD, CUT, false, false, true>(A, st) : lin_go<T, TWO, 64, 256, 1, 4, FWD, CUT>(A, st);
        } else {
            whole ? lin_go<T, TWO, 128, 128, 2, 2, FWD, CUT, false, false, true>(A, st) : lin_go<T, TWO, 128, 128, 2, 2, FWD, CUT>(A, st);
        }
    }
}

}  // namespace gatmi

using namespace gatmi;

extern "C" size_t gatmi_linear_fwd_workspace_bytes(const gatmi_linear *l) {
    if (lin_check(l)) return 0;
    const LinGeom G = lin_geom(l);
    return G.image_f + G.fwd.bytes;
}

extern "C" int gatmi_linear_fwd(const gatmi_linear *l, const void *x, const void *weight, const void *bias,
                                const void *residual, void *y, void *slope, void *ws, size_t ws_bytes, void *stream) {
    if (int e = lin_check(l)) return e;
    if (l->rows == 0) return GATMI_OK;
    GATMI_REQUIRE(x && weight && y, "linear_fwd: null argument");
    const LinGeom G = lin_geom(l);
    const size_t need = G.image_f + G.fwd.bytes;
    if (ws_bytes < need || (need && !ws)) {
        set_error("linear workspace too small: %zu < %zu", ws_bytes, need);
        return GATMI_ERR_WS;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    LinArgs A;
    memset(&A, 0, sizeof(A));
    A.A = x;
    A.B = A.plain = weight;
    A.bias = bias;
    A.res = residual;
    A.C = y;
    A.slope = l->act == GATMI_ACT_NONE ? nullptr : slope;
    A.act = l->act;
    A.M = l->rows;
    A.N = l->out_features;
    A.K = A.ldb = l->in_features;
    A.part = reinterpret_cast<float *>(static_cast<char *>(ws) + G.image_f);
    ProfScope ps("linear_fwd", st);
    if (G.few) {
        GATMI_WITH_TYPE(l->dtype, {
            auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((A.N + 3) / 4), dim3(256), 0, st, A); };
            if (A.M == 1) go(lin_rows_kernel<T, 1>);
            else if (A.M <= 4) go(lin_rows_kernel<T, 4>);
            else go(lin_rows_kernel<T, kFewRows>);
        });
    } else if (G.image_fwd) {
        hipLaunchKernelGGL((lin_image_kernel<float, false>), dim3((G.ldf + 31) / 32, (A.N + 31) / 32), dim3(256), 0, st,
                           static_cast<const float *>(weight), A.N, A.K, G.ldf, ws, nullptr);
        A.B = ws;
        A.ldb = G.ldf;
        lin_launch_nt<float, true, true, false>(A, G.fwd, st);
    } else {
        GATMI_WITH_TYPE(l->dtype, (lin_launch_nt<T, true, false, false>(A, G.fwd, st)));
    }
    GATMI_HIP(hipGetLastError());
    return GATMI_OK;
}

// The backward's workspace: [weights' image][slabs][column sums], the sums of a split dx where the slabs follow
struct LinBwdWs {
    bool one;               // dW's single split writes the gradients themselves
    size_t image, slabs, bytes;
};
static LinBwdWs lin_bwd_ws(const LinGeom &G, bool x, bool w, bool b) {
    LinBwdWs W;
    W.one = G.splits == 1 && w;
    W.image = x ? G.image_b : 0;
    W.slabs = w && !W.one ? G.slabs : 0;
    const size_t dw = W.slabs + (b && !W.one ? G.dbpart : 0), dx = x ? G.dx.bytes : 0;
    W.bytes = W.image + (dw > dx ? dw : dx);
    return W;
}

extern "C" size_t gatmi_linear_bwd_workspace_bytes_of(const gatmi_linear *l, int32_t grad_x, int32_t grad_weight,
                                                      int32_t grad_bias) {
    if (lin_check(l)) return 0;
    return lin_bwd_ws(lin_geom(l), grad_x, grad_weight, grad_bias).bytes;
}

extern "C" size_t gatmi_linear_bwd_workspace_bytes(const gatmi_linear *l) {
    if (lin_check(l)) return 0;
    const LinGeom G = lin_geom(l);
    const size_t all = lin_bwd_ws(G, true, true, true).bytes, some = lin_bwd_ws(G, true, false, true).bytes;
    return all > some ? all : some;
}

extern "C" int gatmi_linear_bwd(const gatmi_linear *l, const void *x, const void *weight, const void *slope,
                                const void *grad_y, void *grad_x, void *grad_weight, void *grad_bias, void *ws,
                                size_t ws_bytes, void *stream) {
    if (int e = lin_check(l)) return e;
    GATMI_REQUIRE(l->rows == 0 || (x && weight && grad_y), "linear_bwd: null argument");
    GATMI_REQUIRE(l->act == GATMI_ACT_NONE || slope || l->rows == 0, "linear_bwd: the activation's slope is missing");
    const LinGeom G = lin_geom(l);
    const LinBwdWs W = lin_bwd_ws(G, grad_x, grad_weight, grad_bias);
    if (ws_bytes < W.bytes || (W.bytes && !ws)) {
        set_error("linear workspace too small: %zu < %zu", ws_bytes, W.bytes);
        return GATMI_ERR_WS;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    char *image = static_cast<char *>(ws);
    float *slabs = reinterpret_cast<float *>(image + W.image), *dbpart = reinterpret_cast<float *>(image + W.image + W.slabs);
    const int N = l->out_features, K = l->in_features;
    LinArgs A;
    memset(&A, 0, sizeof(A));
    A.A = grad_y;
    A.aslope = l->act == GATMI_ACT_NONE ? nullptr : slope;
    A.M = l->rows;
    A.slope_scale = slope_tail_negative(l->act) ? -kSlopeScale : kSlopeScale;
    const bool two = lin_two(l);
    if (grad_x && l->rows > 0) {
        ProfScope ps("linear_dx", st);
        A.plain = weight;
        A.B = image;
        A.C = grad_x;
        A.part = slabs;         // (dW's turn comes after)
        A.N = K;
        A.K = N;
        A.ldb = G.ldb;
        uint8_t *bad = reinterpret_cast<uint8_t *>(image) + (W.image - G.bad_b);
        A.bad = bad;
        A.bad_cols = (G.ldb + 31) / 32;
        GATMI_WITH_TYPE(l->dtype, {
            hipLaunchKernelGGL((lin_image_kernel<T, true>), dim3((G.ldb + 31) / 32, (K + 31) / 32), dim3(256), 0, st,
                               static_cast<const T *>(weight), N, K, G.ldb, ws, two ? bad : nullptr);
            constexpr bool cut = IsF32<T>::value;
            if (two) lin_launch_nt<T, false, cut, !cut>(A, G.dx, st);
            else lin_launch_nt<T, false, cut, false>(A, G.dx, st);
        });
        GATMI_HIP(hipGetLastError());
    }
    if (grad_weight || grad_bias) {
        ProfScope ps("linear_dw", st);
        A.plain = nullptr;
        A.B = x;
        A.N = N;
        A.K = K;
        const bool one = W.one;
        A.part = grad_weight && !one ? slabs : nullptr;
        A.dbpart = grad_bias && !one ? dbpart : nullptr;
        A.dw = one ? grad_weight : nullptr;
        A.db = one ? grad_bias : nullptr;
        A.per_split = G.per_split;
        A.splits = G.splits;
        GATMI_WITH_TYPE(l->dtype, {
            const bool wide = G.wide;
            // (without dW the first column of tiles does: its blocks leave the column sums)
            A.tiles_n = grad_weight ? (K + (wide ? 255 : 127)) / (wide ? 256 : 128) : 1;
            A.tiles = grad_weight ? lin_dw_tiles(l, wide) : (N + kBM - 1) / kBM;
            auto pick = [&](auto t) {
                constexpr bool b = decltype(t)::value;
                return N < 8 || K < 8 ? (wide ? lin_tn_kernel<T, 256, true, b> : lin_tn_kernel<T, 128, true, b>)
                                      : (wide ? lin_tn_kernel<T, 256, false, b> : lin_tn_kernel<T, 128, false, b>);
            };
            auto tn = two ? pick(std::integral_constant<bool, !IsF32<T>::value>{}) : pick(std::false_type{});
            hipLaunchKernelGGL(tn, dim3((unsigned)((A.tiles * G.splits + 7) / 8 * 8)), dim3(wide ? 512 : 256), 0, st, A);
            const long long size = (long long)N * K;
            const int dw_blocks = grad_weight ? (int)((size + 63) / 64) : 0, db_blocks = grad_bias ? (N + 7) / 8 : 0;
            if (!one)
                hipLaunchKernelGGL((lin_slabs_kernel<T>), dim3(dw_blocks + db_blocks), dim3(256), 0, st, slabs, G.splits, size,
                                   static_cast<T *>(grad_weight), dw_blocks, dbpart, N, static_cast<T *>(grad_bias));
        });
        GATMI_HIP(hipGetLastError());
    }
    return GATMI_OK;
}
