// Linear layer with its epilogue:  y = act(x W^T + b) + residual,  and its gradient
//     dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz   (d residual = dy)
// on the matrix cores, in f32, bf16 or f16; every sum is kept in f32.
//
//  * 16-bit tensors multiply as they are (v_mfma_f32_32x32x16_{bf16,f16}).
//  * f32 tensors are cut exactly into three bf16 pieces each, v = p0 + p1 + p2, and multiply as the
//    six products p_i q_j with i + j <= 2: what is left out is 2^-25 of a product, less than an f32
//    multiply rounds, at 16/6 of the f32 MFMA's rate.  A sum that comes out infinite or NaN (an operand
//    was, or a piece rounded up to infinity next to the largest float) is taken again in plain f32.
//  * act'(z) is written by the forward when a backward follows: f32 for f32 tensors, for 16-bit ones as a
//    16-bit fixed-point number of step 2^-15 (0 and 1 are exact), so that dz = dy act'(z) carries one
//    rounding to 16 bits, its own.
#include "attn_device.h"
#include "common.h"
#include "dense_device.h"

namespace gatmi {

typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));
typedef float f32x16v __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes from any element on

// act'(z) in 16 bits: round(d * 2^15) + 2^13, i.e. [-0.25, 1.75); 65535 stands for NaN
__device__ __forceinline__ uint16_t pack_slope(float d) {
    return d != d ? (uint16_t)65535 : (uint16_t)(int)rintf(fmaf(d, 32768.f, 8192.f));
}
__device__ __forceinline__ float unpack_slope(uint16_t q) {
    return q == 65535 ? __uint_as_float(0x7fc00000u) : ((float)(int)q - 8192.f) * (1.0f / 32768.f);
}
template <class T> struct SlopeOf { typedef uint16_t type; };
template <> struct SlopeOf<float> { typedef float type; };
__device__ __forceinline__ float slope_in(float d) { return d; }
__device__ __forceinline__ float slope_in(uint16_t d) { return unpack_slope(d); }
template <class T> __device__ __forceinline__ typename SlopeOf<T>::type slope_out(float d) {
    if constexpr (IsF32<T>::value) return d;
    else return pack_slope(d);
}

// What the kernels need to know of an element type
template <class T> struct Mul;
template <> struct Mul<bf16_t> {
    static constexpr int PIECES = 1, BK = 64;
    static __device__ __forceinline__ f32x16v mma(uint4 a, uint4 b, f32x16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8v, a), __builtin_bit_cast(bf16x8v, b), c, 0, 0, 0);
    }
};
template <> struct Mul<f16_t> {
    static constexpr int PIECES = 1, BK = 64;
    static __device__ __forceinline__ f32x16v mma(uint4 a, uint4 b, f32x16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8v, a), __builtin_bit_cast(f16x8v, b), c, 0, 0, 0);
    }
};
template <> struct Mul<float> {
    static constexpr int PIECES = 3, BK = 32;
    static __device__ __forceinline__ f32x16v mma(uint4 a, uint4 b, f32x16v c) { return Mul<bf16_t>::mma(a, b, c); }
};

// Eight consecutive elements of a row as they lie in memory; `left` of them exist, the rest read as zero
template <class T> struct Gran {
    uint32_t w[2 * sizeof(T)];
};
template <class T> __device__ __forceinline__ Gran<T> ld_gran(const T *p, int left) {
    Gran<T> g;
    if (left >= 8) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
            const u32x4u v = reinterpret_cast<const u32x4u *>(p)[i];
            g.w[4 * i] = v[0]; g.w[4 * i + 1] = v[1]; g.w[4 * i + 2] = v[2]; g.w[4 * i + 3] = v[3];
        }
    } else {
        T e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < left ? p[i] : (T)0.f;
        __builtin_memcpy(g.w, e, sizeof(e));
    }
    return g;
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

// A tile of R rows x BK contraction elements in LDS, PIECES planes of 16-bit elements.  16-byte granules
// are XOR-swizzled so that eight lanes reading one granule column of eight rows hit all banks.
template <class T, int R> struct Tile {
    static constexpr int BK = Mul<T>::BK, G = BK / 8, P = Mul<T>::PIECES;
    static constexpr int PLANE = R * BK * 2, BYTES = PLANE * P;
    static __device__ __forceinline__ int at(int row, int g) {
        const int s = G == 8 ? (row & 7) : ((row >> 1) & 3);
        return row * (BK * 2) + ((g ^ s) << 4);
    }
    static __device__ __forceinline__ void put(char *lds, int row, int g, const Gran<T> &v) {
        if constexpr (P == 1) {
            *reinterpret_cast<uint4 *>(lds + at(row, g)) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
        } else {
            uint32_t q[3][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                cut3(__uint_as_float(v.w[2 * i]), __uint_as_float(v.w[2 * i + 1]), q[0][i], q[1][i], q[2][i]);
#pragma unroll
            for (int p = 0; p < 3; ++p)
                *reinterpret_cast<uint4 *>(lds + p * PLANE + at(row, g)) = make_uint4(q[p][0], q[p][1], q[p][2], q[p][3]);
        }
    }
    // two contraction steps (2m, 2m + 1) of eight rows row0 .. row0 + 7: the transposing store of dW
    static __device__ __forceinline__ void put_pair(char *lds, int row0, int m2, const Gran<T> &lo, const Gran<T> &hi) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int a = at(row0 + i, m2 >> 2) + (m2 & 3) * 4;
            if constexpr (P == 1) {
                const uint32_t l = i & 1 ? lo.w[i / 2] >> 16 : lo.w[i / 2] & 0xffffu;
                const uint32_t h = i & 1 ? hi.w[i / 2] & 0xffff0000u : hi.w[i / 2] << 16;
                *reinterpret_cast<uint32_t *>(lds + a) = l | h;
            } else {
                uint32_t q[3];
                cut3(__uint_as_float(lo.w[i]), __uint_as_float(hi.w[i]), q[0], q[1], q[2]);
#pragma unroll
                for (int p = 0; p < 3; ++p) *reinterpret_cast<uint32_t *>(lds + p * PLANE + a) = q[p];
            }
        }
    }
    static __device__ __forceinline__ uint4 frag(const char *lds, int p, int row, int g) {
        return *reinterpret_cast<const uint4 *>(lds + p * PLANE + at(row, g));
    }
};

struct LinArgs {
    const void *A, *B;        // [M, K] and [N, K], rows of K elements
    const void *bias, *res;
    void *C;                  // [M, N]
    void *slope;              // forward: act'(z) out
    float *part;              // dW: [splits][N][K] slabs
    long long M;
    int N, K;
    long long tiles_n, tiles;
    long long per_split;      // dW: rows of one split
};

constexpr int kBM = 128, kBN = 128;

// acc (32x32 blocks of a wave's 64 x 64) += A-tile rows ra.. x B-tile rows rb..
template <class T> __device__ __forceinline__ void tile_mma(const char *la, const char *lb, int ra, int rb, int lane,
                                                            f32x16v (&acc)[2][2]) {
    typedef Tile<T, kBM> TA;
    typedef Tile<T, kBN> TB;
    const int r = lane & 31, half = lane >> 5;
#pragma unroll
    for (int s = 0; s < TA::BK / 16; ++s) {
        uint4 a[2][TA::P], b[2][TA::P];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int p = 0; p < TA::P; ++p) {
                a[i][p] = TA::frag(la, p, ra + i * 32 + r, 2 * s + half);
                b[i][p] = TB::frag(lb, p, rb + i * 32 + r, 2 * s + half);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if constexpr (TA::P == 1) {
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
}

// row of accumulator register q in a 32 x 32 block (its column is lane & 31)
__device__ __forceinline__ int acc_row(int q, int half) { return (q >> 2) * 8 + half * 4 + (q & 3); }

// C[m][n] = epilogue(sum_k A[m][k] B[n][k]); FWD: bias, activation, residual, slope
template <class T, int ACT, bool FWD>
__global__ __launch_bounds__(256, 2) void lin_nt_kernel(const LinArgs A) {
    typedef Tile<T, kBM> TA;
    typedef Tile<T, kBN> TB;
    constexpr int kLoop = TA::BYTES + TB::BYTES, kEpi = 4 * 32 * 68 * 4;
    __shared__ __attribute__((aligned(16))) char smem[kLoop > kEpi ? kLoop : kEpi];
    char *la = smem, *lb = smem + TA::BYTES;
    // consecutive tiles share rows of A: give each XCD (block index mod 8) a contiguous range of them
    const long long tile = (long long)(blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    if (tile >= A.tiles) return;
    const long long m0 = tile / A.tiles_n * kBM;
    const int n0 = (int)(tile % A.tiles_n) * kBN;
    const T *pa = static_cast<const T *>(A.A), *pb = static_cast<const T *>(A.B);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    constexpr int G = TA::G, NA = kBM * G / 256, NB = kBN * G / 256;
    Gran<T> ga[NA], gb[NB];
    const int g = threadIdx.x % G, row = threadIdx.x / G;
    auto fetch = [&](int k0) {
        const int k = k0 + g * 8;
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            long long m = m0 + row + i * (256 / G);
            if (m >= A.M) m = A.M - 1;             // its results are not stored
            ga[i] = ld_gran<T>(pa + m * A.K + k, A.K - k);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            int n = n0 + row + i * (256 / G);
            if (n >= A.N) n = A.N - 1;
            gb[i] = ld_gran<T>(pb + (long long)n * A.K + k, A.K - k);
        }
    };
    f32x16v acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
    fetch(0);
    for (int k0 = 0; k0 < A.K; k0 += TA::BK) {
#pragma unroll
        for (int i = 0; i < NA; ++i) TA::put(la, row + i * (256 / G), g, ga[i]);
#pragma unroll
        for (int i = 0; i < NB; ++i) TB::put(lb, row + i * (256 / G), g, gb[i]);
        __syncthreads();
        if (k0 + TA::BK < A.K) fetch(k0 + TA::BK);
        tile_mma<T>(la, lb, wm, wn, lane, acc);
        __syncthreads();
    }
    // epilogue: a wave turns its blocks 32 rows at a time through LDS of its own into row pieces of 8
    constexpr int LD = 68;
    float *le = reinterpret_cast<float *>(smem) + wave * 32 * LD;
    const int half = lane >> 5, c8 = (lane & 7) * 8, r8 = lane >> 3;
    const int n = n0 + wn + c8;
    const int have = A.N - n;                       // columns of this piece that exist
    float bias[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
        bias[k] = FWD && A.bias && k < have ? (float)static_cast<const T *>(A.bias)[n + k] : 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) le[acc_row(q, half) * LD + j * 32 + (lane & 31)] = acc[i][j][q];
        __syncthreads();
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const long long m = m0 + wm + i * 32 + p * 8 + r8;
            if (m >= A.M || have <= 0) continue;
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = le[(p * 8 + r8) * LD + c8 + k];
            if constexpr (IsF32<T>::value) {        // see the head of this file
                bool fine = true;
#pragma unroll
                for (int k = 0; k < 8; ++k) fine = fine && fabsf(v[k]) < INFINITY;
                if (!fine)
                    for (int k = 0; k < 8; ++k) {
                        if (k >= have || fabsf(v[k]) < INFINITY) continue;
                        float s = 0.f;
                        for (int kk = 0; kk < A.K; ++kk)
                            s = fmaf((float)pa[m * A.K + kk], (float)pb[(long long)(n + k) * A.K + kk], s);
                        v[k] = s;
                    }
            }
            const long long at = m * A.N + n;
            T *out = static_cast<T *>(A.C) + at;
            const T *res = static_cast<const T *>(A.res) + at;
            typedef typename SlopeOf<T>::type ST;
            ST *so = static_cast<ST *>(A.slope) + at;
            if (have >= 8) {
                VecF<8> o, rr;
                ST sl[8];
                if (FWD && A.res) rr = ldv<T, 8>(res);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    float y = v[k];
                    if constexpr (FWD) {
                        float d;
                        y = act_both<ACT, IsF32<T>::value>(y + bias[k], d);
                        sl[k] = slope_out<T>(d);
                        if (A.res) y += rr.e[k];
                    }
                    o.e[k] = y;
                }
                stv<T, 8>(out, o);
                if (FWD && ACT != GATMI_ACT_NONE && A.slope) {
#pragma unroll
                    for (int w = 0; w < (int)sizeof(ST) / 2; ++w) {
                        u32x4u t;
                        __builtin_memcpy(&t, sl + w * (16 / sizeof(ST)), 16);
                        reinterpret_cast<u32x4u *>(so)[w] = t;
                    }
                }
            } else {
                for (int k = 0; k < 8; ++k) {
                    if (k >= have) break;
                    float y = v[k];
                    if constexpr (FWD) {
                        float d;
                        y = act_both<ACT, IsF32<T>::value>(y + bias[k], d);
                        if (ACT != GATMI_ACT_NONE && A.slope) so[k] = slope_out<T>(d);
                        if (A.res) y += (float)res[k];
                    }
                    out[k] = (T)y;
                }
            }
        }
    }
}

// dW slabs: part[split][n][k] = sum over the split's rows of A[m][n] B[m][k]  (A = dz [M, N], B = x [M, K])
template <class T> __global__ __launch_bounds__(256, 2) void lin_tn_kernel(const LinArgs A) {
    typedef Tile<T, kBM> TA;
    typedef Tile<T, kBN> TB;
    __shared__ __attribute__((aligned(16))) char smem[TA::BYTES + TB::BYTES];
    char *la = smem, *lb = smem + TA::BYTES;
    const long long split = blockIdx.x / A.tiles;
    const int tile = (int)(blockIdx.x - split * A.tiles);
    const int n0 = tile / (int)A.tiles_n * kBM, k0 = tile % (int)A.tiles_n * kBN;
    const long long r0 = split * A.per_split, r1 = r0 + A.per_split < A.M ? r0 + A.per_split : A.M;
    const T *pa = static_cast<const T *>(A.A), *pb = static_cast<const T *>(A.B);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    // a thread's pieces: contraction pair (2 * pr, + 1), eight channels ch ..
    constexpr int PAIRS = TA::BK / 2, GC = 256 / PAIRS, NP = kBM / 8 / GC;
    const int pr = threadIdx.x % PAIRS, cg = threadIdx.x / PAIRS;
    Gran<T> ga[NP][2], gb[NP][2];
    auto fetch = [&](long long r) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const long long m = r + 2 * pr + u;
                const bool in = m < r1;
                const int ca = n0 + (cg + i * GC) * 8, cb = k0 + (cg + i * GC) * 8;
                ga[i][u] = ld_gran<T>(pa + (in ? m : r0) * A.N + (ca < A.N ? ca : 0), in ? A.N - ca : 0);
                gb[i][u] = ld_gran<T>(pb + (in ? m : r0) * A.K + (cb < A.K ? cb : 0), in ? A.K - cb : 0);
            }
    };
    f32x16v acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
    if (r0 < r1) fetch(r0);
    for (long long r = r0; r < r1; r += TA::BK) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            TA::put_pair(la, (cg + i * GC) * 8, pr, ga[i][0], ga[i][1]);
            TB::put_pair(lb, (cg + i * GC) * 8, pr, gb[i][0], gb[i][1]);
        }
        __syncthreads();
        if (r + TA::BK < r1) fetch(r + TA::BK);
        tile_mma<T>(la, lb, wm, wn, lane, acc);
        __syncthreads();
    }
    float *part = A.part + split * (long long)A.N * A.K;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                const int n = n0 + wm + i * 32 + acc_row(q, lane >> 5), k = k0 + wn + j * 32 + (lane & 31);
                if (n >= A.N || k >= A.K) continue;
                float v = acc[i][j][q];
                if (IsF32<T>::value && !(fabsf(v) < INFINITY)) {
                    v = 0.f;
                    for (long long m = r0; m < r1; ++m) v = fmaf((float)pa[m * A.N + n], (float)pb[m * A.K + k], v);
                }
                part[(long long)n * A.K + k] = v;
            }
}

// dW = sum of the slabs, in order
template <class T> __global__ __launch_bounds__(256) void lin_slabs_kernel(const float *part, int splits, long long size, T *out) {
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < size; i += gridDim.x * 256ll) {
        float s = 0.f;
        for (int q = 0; q < splits; ++q) s += part[q * size + i];
        out[i] = (T)s;
    }
}

// dz = dy * act'(z) (DZ: written), and its column sums per block (part [blocks][N], when part)
template <class T, int V, bool DZ>
__global__ __launch_bounds__(256) void lin_dz_kernel(const T *dy, const typename SlopeOf<T>::type *slope, T *dz,
                                                     float *part, long long rows, int N) {
    __shared__ VecF<V> red[256];
    const int nslot = (N + V - 1) / V, first = blockIdx.y * 256;
    const int slots = nslot - first < 256 ? nslot - first : 256;
    const int rpp = 256 / slots, s = threadIdx.x % slots, rsub = threadIdx.x / slots;
    const int j = (first + s) * V, off = j + V <= N ? j : N - V, skip = j - off;
    const long long per = (rows + gridDim.x - 1) / gridDim.x, r0 = blockIdx.x * per, r1 = r0 + per < rows ? r0 + per : rows;
    VecF<V> sum;
#pragma unroll
    for (int k = 0; k < V; ++k) sum.e[k] = 0.f;
    if (rsub < rpp)
#pragma unroll 4
        for (long long r = r0 + rsub; r < r1; r += rpp) {
            VecF<V> g = ldv<T, V>(dy + r * N + off);
            if (DZ) {
                typename SlopeOf<T>::type q[V];
                __builtin_memcpy(q, slope + r * N + off, sizeof(q));
#pragma unroll
                for (int k = 0; k < V; ++k) g.e[k] *= slope_in(q[k]);
                stv<T, V>(dz + r * N + off, g);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) sum.e[k] += g.e[k];
        }
    if (!part) return;
    red[threadIdx.x] = sum;
    __syncthreads();
    if ((int)threadIdx.x < slots) {
        for (int q = 1; q < rpp; ++q)
#pragma unroll
            for (int k = 0; k < V; ++k) sum.e[k] += red[threadIdx.x + q * slots].e[k];
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k >= skip) part[(long long)blockIdx.x * N + off + k] = sum.e[k];
    }
}
template <class T> __global__ __launch_bounds__(256) void lin_db_kernel(const float *part, int blocks, int N, T *db) {
    __shared__ double red[256];
    const int c = blockIdx.x * 8 + (threadIdx.x & 7), rg = threadIdx.x >> 3;
    double s = 0.0;
    if (c < N)
        for (int b = rg; b < blocks; b += 32) s += part[(long long)b * N + c];
    red[threadIdx.x] = s;
    __syncthreads();
    if (rg == 0 && c < N) {
        for (int q = 1; q < 32; ++q) s += red[threadIdx.x + q * 8];
        db[c] = (T)(float)s;
    }
}

// out[k][n] = w[n][k]
template <class T> __global__ __launch_bounds__(256) void lin_transpose_kernel(const T *w, int N, int K, T *out) {
    __shared__ T t[32][33];
    const int k0 = blockIdx.x * 32, n0 = blockIdx.y * 32, x = threadIdx.x & 31, y = threadIdx.x >> 5;
    for (int i = y; i < 32; i += 8)
        if (n0 + i < N && k0 + x < K) t[i][x] = w[(long long)(n0 + i) * K + k0 + x];
    __syncthreads();
    for (int i = y; i < 32; i += 8)
        if (k0 + i < K && n0 + x < N) out[(long long)(k0 + i) * N + n0 + x] = t[x][i];
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

constexpr int kDzBlocks = 2048;
struct LinGeom {
    int dz_blocks, splits;
    long long per_split;
    size_t dz, wt, part, slabs;     // bytes
};
static LinGeom lin_geom(const gatmi_linear *l) {
    LinGeom G;
    const size_t el = l->dtype == GATMI_F32 ? 4 : 2;
    const long long b = (l->rows + 31) / 32;
    G.dz_blocks = (int)(b < 1 ? 1 : (b > kDzBlocks ? kDzBlocks : b));
    const long long tiles = ((l->out_features + kBM - 1ll) / kBM) * ((l->in_features + kBN - 1ll) / kBN);
    // enough splits of the rows for two blocks a CU, at least 256 rows each
    long long s = (2ll * device_cus() + tiles - 1) / tiles;
    const long long most = (l->rows + 255) / 256;
    if (s > most) s = most;
    if (s < 1) s = 1;
    const int bk = l->dtype == GATMI_F32 ? 32 : 64;
    G.per_split = ((l->rows + s - 1) / s + bk - 1) / bk * bk;
    if (G.per_split < bk) G.per_split = bk;
    G.splits = (int)((l->rows + G.per_split - 1) / G.per_split);
    if (G.splits < 1) G.splits = 1;
    G.dz = align_up((size_t)l->rows * l->out_features * el);
    G.wt = align_up((size_t)l->in_features * l->out_features * el);
    G.part = align_up((size_t)G.dz_blocks * l->out_features * 4);
    G.slabs = align_up((size_t)G.splits * l->in_features * l->out_features * 4);
    return G;
}

template <class T> static void lin_launch_nt(LinArgs A, bool fwd, int act, hipStream_t st) {
    A.tiles_n = (A.N + kBN - 1) / kBN;
    A.tiles = (A.M + kBM - 1) / kBM * A.tiles_n;
    const unsigned grid = (unsigned)((A.tiles + 7) / 8 * 8);
    if (!fwd) {
        hipLaunchKernelGGL((lin_nt_kernel<T, GATMI_ACT_NONE, false>), dim3(grid), dim3(256), 0, st, A);
        return;
    }
    GATMI_WITH_ACT(act, hipLaunchKernelGGL((lin_nt_kernel<T, ACT, true>), dim3(grid), dim3(256), 0, st, A));
}

}  // namespace gatmi

using namespace gatmi;

extern "C" int gatmi_linear_fwd(const gatmi_linear *l, const void *x, const void *weight, const void *bias,
                                const void *residual, void *y, void *slope, void *stream) {
    if (int e = lin_check(l)) return e;
    if (l->rows == 0) return GATMI_OK;
    GATMI_REQUIRE(x && weight && y, "linear_fwd: null argument");
    hipStream_t st = static_cast<hipStream_t>(stream);
    LinArgs A;
    memset(&A, 0, sizeof(A));
    A.A = x;
    A.B = weight;
    A.bias = bias;
    A.res = residual;
    A.C = y;
    A.slope = slope;
    A.M = l->rows;
    A.N = l->out_features;
    A.K = l->in_features;
    ProfScope ps("linear_fwd", st);
    GATMI_WITH_TYPE(l->dtype, lin_launch_nt<T>(A, true, l->act, st));
    GATMI_HIP(hipGetLastError());
    return GATMI_OK;
}

extern "C" size_t gatmi_linear_bwd_workspace_bytes(const gatmi_linear *l) {
    if (lin_check(l)) return 0;
    const LinGeom G = lin_geom(l);
    return G.dz + G.wt + G.part + G.slabs + 256;
}

extern "C" int gatmi_linear_bwd(const gatmi_linear *l, const void *x, const void *weight, const void *slope,
                                const void *grad_y, void *grad_x, void *grad_weight, void *grad_bias, void *ws,
                                size_t ws_bytes, void *stream) {
    if (int e = lin_check(l)) return e;
    GATMI_REQUIRE(l->rows == 0 || (x && weight && grad_y), "linear_bwd: null argument");
    GATMI_REQUIRE(l->act == GATMI_ACT_NONE || slope || l->rows == 0, "linear_bwd: the activation's slope is missing");
    const LinGeom G = lin_geom(l);
    if (!ws || ws_bytes < G.dz + G.wt + G.part + G.slabs) {
        set_error("linear workspace too small: %zu < %zu", ws_bytes, G.dz + G.wt + G.part + G.slabs);
        return GATMI_ERR_WS;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    char *base = static_cast<char *>(ws);
    const int N = l->out_features, K = l->in_features;
    const bool has_act = l->act != GATMI_ACT_NONE;
    float *part = reinterpret_cast<float *>(base + G.dz + G.wt), *slabs = reinterpret_cast<float *>(base + G.dz + G.wt + G.part);
    const void *dz = has_act ? base : grad_y;
    if (l->rows > 0 && (has_act || grad_bias)) {
        ProfScope ps("linear_dz", st);
        GATMI_WITH_TYPE(l->dtype, {
            constexpr int VM = 16 / sizeof(T);
            const int v = N >= VM ? VM : (N >= 4 && VM == 8 ? 4 : (N >= 2 ? 2 : 1));
            const dim3 grid(G.dz_blocks, ((N + v - 1) / v + 255) / 256);
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, static_cast<const T *>(grad_y),
                                   static_cast<const typename SlopeOf<T>::type *>(slope), reinterpret_cast<T *>(base),
                                   grad_bias ? part : nullptr, (long long)l->rows, N);
            };
            if (has_act) {
                if (v == VM) go(lin_dz_kernel<T, VM, true>);
                else if (v == 4) go(lin_dz_kernel<T, 4, true>);
                else if (v == 2) go(lin_dz_kernel<T, 2, true>);
                else go(lin_dz_kernel<T, 1, true>);
            } else {
                if (v == VM) go(lin_dz_kernel<T, VM, false>);
                else if (v == 4) go(lin_dz_kernel<T, 4, false>);
                else if (v == 2) go(lin_dz_kernel<T, 2, false>);
                else go(lin_dz_kernel<T, 1, false>);
            }
        });
        GATMI_HIP(hipGetLastError());
    }
    if (grad_bias) {
        ProfScope ps("linear_db", st);
        GATMI_WITH_TYPE(l->dtype, hipLaunchKernelGGL((lin_db_kernel<T>), dim3((N + 7) / 8), dim3(256), 0, st, part,
                                                     l->rows > 0 ? G.dz_blocks : 0, N, static_cast<T *>(grad_bias)));
        GATMI_HIP(hipGetLastError());
    }
    if (grad_x && l->rows > 0) {
        ProfScope ps("linear_dx", st);
        GATMI_WITH_TYPE(l->dtype, {
            T *wt = reinterpret_cast<T *>(base + G.dz);
            hipLaunchKernelGGL((lin_transpose_kernel<T>), dim3((K + 31) / 32, (N + 31) / 32), dim3(256), 0, st,
                               static_cast<const T *>(weight), N, K, wt);
            LinArgs A;
            memset(&A, 0, sizeof(A));
            A.A = dz;
            A.B = wt;
            A.C = grad_x;
            A.M = l->rows;
            A.N = K;
            A.K = N;
            lin_launch_nt<T>(A, false, GATMI_ACT_NONE, st);
        });
        GATMI_HIP(hipGetLastError());
    }
    if (grad_weight) {
        ProfScope ps("linear_dw", st);
        GATMI_WITH_TYPE(l->dtype, {
            LinArgs A;
            memset(&A, 0, sizeof(A));
            A.A = dz;
            A.B = x;
            A.M = l->rows;
            A.N = N;
            A.K = K;
            A.part = slabs;
            A.tiles_n = (K + kBN - 1) / kBN;
            A.tiles = (long long)((N + kBM - 1) / kBM) * A.tiles_n;
            A.per_split = G.per_split;
            hipLaunchKernelGGL((lin_tn_kernel<T>), dim3((unsigned)(A.tiles * G.splits)), dim3(256), 0, st, A);
            const long long size = (long long)N * K;
            const long long b = (size + 255) / 256;
            hipLaunchKernelGGL((lin_slabs_kernel<T>), dim3((unsigned)(b > 4096 ? 4096 : b)), dim3(256), 0, st, slabs,
                               G.splits, size, static_cast<T *>(grad_weight));
        });
        GATMI_HIP(hipGetLastError());
    }
    return GATMI_OK;
}
