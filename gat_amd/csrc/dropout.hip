// Dropout as an operator of its own: y = keep ? x / (1 - p) : 0, + residual.  The keep decision is the
// counter hash of (seed, row, column) that the fused glue uses (attn_device.h), so nothing is stored:
// the backward draws the same decisions again from the seed.
//
// One pass over a flat array; 16 bytes per lane and access whatever the row width, the (row, column) of a
// vector's first element from one multiply-high division, the following ones by counting.  Memory bounds it:
// [2449029, 100] bf16 with a residual in 287 us (1.47 GB, 5.1 TB/s), its backward in 214 us (0.98 GB, 4.6 TB/s).
#include "attn_device.h"
#include "common.h"
#include "dense_device.h"

namespace gatmi {

constexpr int kDropUnroll = 4;
constexpr int kDropBlocks = 4096;

struct DropArgs {
    const void *x, *res;
    void *y;
    long long total;          // rows * cols
    FastDiv cols;
    uint32_t thr, seed_lo, seed_hi;
    float inv_keep;
    const uint64_t *seed_dev; // read here when set
    uint64_t *seed_used;      // receives the seed (the backward's, when the caller's moves on)
    long long step_row;       // grid stride in (rows, columns)
    uint32_t step_col;
};

// res is read only when RES; WRAP: a vector can span two rows
template <class T, bool RES, bool WRAP>
__global__ __launch_bounds__(256) void dropout_kernel(const DropArgs A) {
    constexpr int V = 16 / sizeof(T);
    constexpr int kChunk = 256 * V * kDropUnroll;
    uint32_t lo = A.seed_lo, hi = A.seed_hi;
    if (A.seed_dev) {
        const uint64_t s = *A.seed_dev;
        lo = (uint32_t)s;
        hi = (uint32_t)(s >> 32);
    }
    if (A.seed_used && blockIdx.x == 0 && threadIdx.x == 0) *A.seed_used = ((uint64_t)hi << 32) | lo;
    const T *x = static_cast<const T *>(A.x), *res = static_cast<const T *>(A.res);
    T *y = static_cast<T *>(A.y);
    const uint32_t cols = A.cols.d;
    const long long first = (long long)blockIdx.x * kChunk;
    uint32_t row0 = (uint32_t)(first / cols), col0 = (uint32_t)(first % cols);
    for (long long base = first; base < A.total; base += (long long)gridDim.x * kChunk) {
        VecF<V> v[kDropUnroll], r[kDropUnroll];
#pragma unroll
        for (int u = 0; u < kDropUnroll; ++u) {
            const long long i = base + (u * 256 + threadIdx.x) * V;
            if (i + V <= A.total) {
                v[u] = ldv<T, V>(x + i);
                if (RES) r[u] = ldv<T, V>(res + i);
            } else {
                for (int k = 0; k < V; ++k) {
                    v[u].e[k] = i + k < A.total ? (float)x[i + k] : 0.f;
                    if (RES) r[u].e[k] = i + k < A.total ? (float)res[i + k] : 0.f;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kDropUnroll; ++u) {
            const uint32_t off = (u * 256 + threadIdx.x) * V;
            const long long i = base + off;
            const uint32_t c = col0 + off;            // < 2^31 + a chunk
            const uint32_t q = fdiv(A.cols, c);
            uint32_t col = c - q * cols;
            // the two products of keep_hash's first line, advanced by addition from element to element
            uint32_t a = (row0 + q) * 0x9E3779B1u + lo, b = col * 0x85EBCA77u + hi;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                uint32_t h = a ^ b;
                h ^= h >> 15; h *= 0x2C1B3C6Du; h ^= h >> 12; h *= 0x297A2D39u; h ^= h >> 15;
                float o = (h >> 8) >= A.thr ? v[u].e[k] * A.inv_keep : 0.f;
                if (RES) o += r[u].e[k];
                v[u].e[k] = o;
                b += 0x85EBCA77u;
                if (WRAP && ++col == cols) {
                    col = 0;
                    b = hi;
                    a += 0x9E3779B1u;
                }
            }
            if (i + V <= A.total) {
                stv<T, V>(y + i, v[u]);
            } else {
                for (int k = 0; k < V; ++k)
                    if (i + k < A.total) y[i + k] = (T)v[u].e[k];
            }
        }
        row0 += (uint32_t)A.step_row;
        col0 += A.step_col;
        if (col0 >= cols) {
            col0 -= cols;
            ++row0;
        }
    }
}

}  // namespace gatmi

using namespace gatmi;

extern "C" int gatmi_dropout(int32_t dtype, int64_t rows, int64_t cols, float dropout_p, uint64_t seed,
                             const uint64_t *seed_on_device, uint64_t *seed_used, const void *x,
                             const void *residual, void *y, void *stream) {
    GATMI_REQUIRE(dtype >= GATMI_F32 && dtype <= GATMI_F16, "dropout: unknown element type %d", dtype);
    GATMI_REQUIRE(rows >= 0 && rows < (1ll << 32) && cols >= 1 && cols < (1ll << 31),
                  "dropout: rows %lld / cols %lld out of range", (long long)rows, (long long)cols);
    GATMI_REQUIRE(dropout_p >= 0.f && dropout_p < 1.f, "dropout: p %f outside [0,1)", dropout_p);
    GATMI_REQUIRE(rows == 0 || (x && y), "dropout: null argument");
    if (rows == 0 && !seed_used) return GATMI_OK;
    hipStream_t st = static_cast<hipStream_t>(stream);
    DropArgs A;
    memset(&A, 0, sizeof(A));
    A.x = x;
    A.res = residual;
    A.y = y;
    A.total = rows * cols;
    A.cols = make_fast_div((uint32_t)cols);
    A.thr = (uint32_t)((double)dropout_p * 16777216.0);
    A.seed_lo = (uint32_t)seed;
    A.seed_hi = (uint32_t)(seed >> 32);
    A.inv_keep = 1.0f / (1.0f - dropout_p);
    A.seed_dev = seed_on_device;
    A.seed_used = seed_used;
    ProfScope ps("dropout", st);
    GATMI_WITH_TYPE(dtype, {
        constexpr int V = 16 / sizeof(T);
        constexpr long long kChunk = 256ll * V * kDropUnroll;
        long long blocks = (A.total + kChunk - 1) / kChunk;
        blocks = blocks < 1 ? 1 : (blocks > kDropBlocks ? kDropBlocks : blocks);
        A.step_row = blocks * kChunk / cols;
        A.step_col = (uint32_t)(blocks * kChunk % cols);
        const bool wrap = cols % V != 0;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, A); };
        if (residual)
            wrap ? go(dropout_kernel<T, true, true>) : go(dropout_kernel<T, true, false>);
        else
            wrap ? go(dropout_kernel<T, false, true>) : go(dropout_kernel<T, false, false>);
    });
    GATMI_HIP(hipGetLastError());
    return GATMI_OK;
}
