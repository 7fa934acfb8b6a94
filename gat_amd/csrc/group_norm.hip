// Group normalisation with an activation, channels last: x [batch, length, C], C = groups * width,
//     xh = (x - mean) * rstd   mean / variance over (length, width) of one sample's group
//     y  = act(w xh + b)
// and its gradient, with u = w xh + b, du = dy act'(u), g = w du:
//     dw = sum du xh,  db = sum du,  dx = rstd (g - mean(g) - xh mean(g xh))
//
// Two forms, by what a group is in memory:
//   length == 1 (one node per sample): a sample's group is `width` CONTIGUOUS elements, so the tensor is
//     one list of batch * groups segments.  W lanes own a segment, hold it in registers, and read
//     it once: mean, centred variance and the result come from the same registers.
//   length > 1: a block owns a range of a sample's positions and keeps its lanes on fixed channels;
//     per-channel means and squares around them, joined with Chan's formula (the blocks' in double), then a pass
//     that applies them.
// No sum is made with atomics: the same inputs give the same bits.
//
// Memory bounds all of it.  [100000, 8 x 30] f32: forward with the statistics kept 36 us for 193 MB (5.3 TB/s),
// backward 49 us for 289 MB (5.9 TB/s) and 10 us for the parameter sums.  [3, 169343, 256] bf16: statistics 67 us
// (260 MB), applying them 85 (520 MB), the backward's sums 136 (520 MB), dx 139 (780 MB, 5.6 TB/s); the sums'
// pass is the one that its arithmetic holds back (SiLU and its derivative for two bytes read of x), and x and dy
// are read twice because a sample of 87 MB fits no block's memory.
#include "attn_device.h"
#include "common.h"
#include "dense_device.h"

namespace gatmi {

constexpr int kGnMaxT = 8;         // vectors per lane of the segment kernels
constexpr int kGnFwdBlocks = 4096, kGnBwdBlocks = 1024;
// Blocks of the length > 1 form, over all samples: of the passes that leave sums (each block's are read again)
// and of those that only apply.  Twelve blocks a CU for the sums: 158 -> 137 us for the backward's at
// [3, 169343, 256] bf16 against six; the forward's does not care.
constexpr int kGnChunks = 12 * 256, kGnApply = 24 * 256;
constexpr int kGnJoin = 1024;      // most threads of a block that joins a group's chunks
constexpr int kGnSamples = 65535;  // samples of one launch
constexpr int kGnSlabs = 64;       // row slabs of the column sums

struct GnArgs {
    const void *x, *dy, *w, *b;
    void *y, *dx, *dw, *db;
    float *mean, *rstd;     // [batch, groups]
    float *part;            // segment kernels: [2][slots][width]; chunk kernels: [batch][chunks][2][C]
    float *coef;            // chunk kernels, backward: [batch][groups][2]
    long long nseg;         // batch * groups
    long long length;
    int groups, width, C, chunks, W, w_log;
    float eps, inv_n;
};

// Sum over W consecutive lanes (a power of two); every lane gets it
__device__ __forceinline__ float lanes_sum(float v, int W) {
    for (int o = 1; o < W; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// A lane's vectors of a segment: vector t starts at element (t * W + lane) * V, stepped back to
// width - V where it would run over the end; its first `skip` elements are then another lane's.
template <int V> struct SegSlot {
    int off, skip;      // skip = V: nothing here
};
template <int V> __device__ __forceinline__ SegSlot<V> seg_slot(int t, int W, int lane, int width) {
    const int j = (t * W + lane) * V;
    SegSlot<V> s;
    if (j >= width) {
        s.off = 0;
        s.skip = V;
    } else {
        s.off = j + V <= width ? j : width - V;
        s.skip = j - s.off;
    }
    return s;
}

// ---- length == 1 -----------------------------------------------------------------------------
template <class T, int V, int TT, int ACT, bool SAVE>
__global__ __launch_bounds__(256) void gn_seg_fwd_kernel(const GnArgs A) {
    const int lane = threadIdx.x & (A.W - 1);
    const int per_block = 256 >> A.w_log;
    const T *x = static_cast<const T *>(A.x);
    T *y = static_cast<T *>(A.y);
    const T *gw = static_cast<const T *>(A.w), *gb = static_cast<const T *>(A.b);
    SegSlot<V> sl[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) sl[t] = seg_slot<V>(t, A.W, lane, A.width);
    // the grid's stride is a multiple of `groups` (launcher), so a lane keeps its channels
    const long long seg0 = (long long)blockIdx.x * per_block + (threadIdx.x >> A.w_log);
    const int c0 = (int)(seg0 % A.groups) * A.width;
    VecF<V> w[TT], b[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        w[t] = ldv<T, V>(gw + c0 + sl[t].off);
        b[t] = ldv<T, V>(gb + c0 + sl[t].off);
    }
    const long long stride = (long long)gridDim.x * per_block;
    for (long long seg = seg0; seg < A.nseg; seg += stride) {
        const T *xp = x + seg * A.width;
        VecF<V> v[TT];
        float s = 0.f;
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            v[t] = ldv<T, V>(xp + sl[t].off);
#pragma unroll
            for (int k = 0; k < V; ++k) s += k >= sl[t].skip ? v[t].e[k] : 0.f;
        }
        const float mean = lanes_sum(s, A.W) * A.inv_n;
        float q = 0.f;
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = v[t].e[k] - mean;
                v[t].e[k] = d;
                q += k >= sl[t].skip ? d * d : 0.f;
            }
        const float rstd = 1.0f / sqrtf(lanes_sum(q, A.W) * A.inv_n + A.eps);
        if (SAVE && lane == 0) {
            A.mean[seg] = mean;
            A.rstd[seg] = rstd;
        }
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            if (sl[t].skip == V) continue;
#pragma unroll
            for (int k = 0; k < V; ++k)
                v[t].e[k] = act_value<ACT, IsF32<T>::value>(fmaf(v[t].e[k] * rstd, w[t].e[k], b[t].e[k]));
            stv<T, V>(y + seg * A.width + sl[t].off, v[t]);   // overlapping lanes store equal values
        }
    }
}

// part: [2][slots][width], slot = a lane group of the grid; slot % groups is its group
template <class T, int V, int TT, int ACT>
__global__ __launch_bounds__(256) void gn_seg_bwd_kernel(const GnArgs A) {
    const int lane = threadIdx.x & (A.W - 1);
    const int per_block = 256 >> A.w_log;
    const T *x = static_cast<const T *>(A.x), *dy = static_cast<const T *>(A.dy);
    T *dx = static_cast<T *>(A.dx);
    const T *gw = static_cast<const T *>(A.w), *gb = static_cast<const T *>(A.b);
    SegSlot<V> sl[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) sl[t] = seg_slot<V>(t, A.W, lane, A.width);
    const long long seg0 = (long long)blockIdx.x * per_block + (threadIdx.x >> A.w_log);
    const int c0 = (int)(seg0 % A.groups) * A.width;
    VecF<V> w[TT], b[TT], sw[TT], sb[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        w[t] = ldv<T, V>(gw + c0 + sl[t].off);
        b[t] = ldv<T, V>(gb + c0 + sl[t].off);
#pragma unroll
        for (int k = 0; k < V; ++k) sw[t].e[k] = sb[t].e[k] = 0.f;
    }
    const long long stride = (long long)gridDim.x * per_block;
    for (long long seg = seg0; seg < A.nseg; seg += stride) {
        const float mean = A.mean[seg], rstd = A.rstd[seg];
        VecF<V> h[TT], g[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            h[t] = ldv<T, V>(x + seg * A.width + sl[t].off);
            g[t] = ldv<T, V>(dy + seg * A.width + sl[t].off);
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int t = 0; t < TT; ++t)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float xh = (h[t].e[k] - mean) * rstd;
                float d;
                act_both<ACT, IsF32<T>::value>(fmaf(xh, w[t].e[k], b[t].e[k]), d);
                const bool mine = k >= sl[t].skip;
                const float du = g[t].e[k] * d;
                if (mine) {
                    sb[t].e[k] += du;
                    sw[t].e[k] = fmaf(du, xh, sw[t].e[k]);
                }
                const float gu = du * w[t].e[k];
                h[t].e[k] = xh;
                g[t].e[k] = gu;
                s1 += mine ? gu : 0.f;
                s2 += mine ? gu * xh : 0.f;
            }
        s1 = lanes_sum(s1, A.W) * A.inv_n;
        s2 = lanes_sum(s2, A.W) * A.inv_n;
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            if (sl[t].skip == V) continue;
#pragma unroll
            for (int k = 0; k < V; ++k) g[t].e[k] = rstd * (g[t].e[k] - s1 - h[t].e[k] * s2);
            stv<T, V>(dx + seg * A.width + sl[t].off, g[t]);
        }
    }
    float *pw = A.part + seg0 * A.width, *pb = pw + stride * A.width;
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k >= sl[t].skip) {
                pw[sl[t].off + k] = sw[t].e[k];
                pb[sl[t].off + k] = sb[t].e[k];
            }
}

// ---- length > 1 ------------------------------------------------------------------------------
// Thread -> (channel vector, row offset): lanes of a row side by side, `rpp` rows at a time.  Rows wider
// than 256 vectors are walked in column blocks (blockIdx.z).  A vector that would run over the row's end
// steps back, as above.
struct GnLay {
    int off, skip, rsub, rpp, slots;
    bool on;
    long long r0, r1;
};
template <int V> __device__ __forceinline__ GnLay gn_lay(const GnArgs &A) {
    GnLay L;
    const int nslot = (A.C + V - 1) / V;
    const int first = blockIdx.z * 256;
    L.slots = nslot - first < 256 ? nslot - first : 256;
    L.rpp = 256 / L.slots;
    const int s = threadIdx.x % L.slots;
    L.rsub = threadIdx.x / L.slots;
    L.on = L.rsub < L.rpp;
    const int j = (first + s) * V;
    L.off = j + V <= A.C ? j : A.C - V;
    L.skip = j - L.off;
    const long long per = (A.length + A.chunks - 1) / A.chunks;
    L.r0 = (long long)blockIdx.x * per;
    L.r1 = L.r0 + per < A.length ? L.r0 + per : A.length;
    return L;
}

// per (sample, chunk, channel): mean and M2 of its rows -> part.  A lane takes kGnRows rows at once, their mean and
// the squares around it, and folds them into what it has by Chan's formula, as the lanes are folded in the end: no
// step subtracts large squares from each other, whatever the rows are.  (Sums of d and d^2 with d counted from the
// chunk's first row are as short, but lose log2(rows) digits of the variance when that row is an outlier.)  Everything
// is counted from a value of the chunk, the middle one of three rows' (at a fifth, three and six sevenths: not where
// blocks of data begin), which keeps a mean far from 0 out of the rounding, and an outlier too.  FEW: up to kGnFew rows
// a chunk, where those sums lose no more than kGnFew f32 steps of the variance and need one barrier and half the
// registers: [100000, 4, 64] f32 forward 368 us, 429 without.
constexpr int kGnRows = 8, kGnFew = 64;
template <class T, int V, bool FEW> __global__ __launch_bounds__(256) void gn_stats_kernel(const GnArgs A) {
    __shared__ VecF<V> red[2][256];
    __shared__ float count[256];
    const GnLay L = gn_lay<V>(A);
    const T *x = static_cast<const T *>(A.x) + (long long)blockIdx.y * A.length * A.C + L.off;
    VecF<V> mean, m2, sh;
#pragma unroll
    for (int k = 0; k < V; ++k) mean.e[k] = m2.e[k] = sh.e[k] = 0.f;
    const long long rows = L.r1 - L.r0;
    float *p = A.part + ((long long)blockIdx.y * A.chunks + blockIdx.x) * 2 * A.C + L.off;
    if constexpr (FEW) {
        if (rows > 0) sh = ldv<T, V>(x + L.r0 * A.C);
        if (L.on)
#pragma unroll 4
            for (long long r = L.r0 + L.rsub; r < L.r1; r += L.rpp) {
                const VecF<V> v = ldv<T, V>(x + r * A.C);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float d = v.e[k] - sh.e[k];
                    mean.e[k] += d;
                    m2.e[k] = fmaf(d, d, m2.e[k]);
                }
            }
        red[0][threadIdx.x] = mean;
        red[1][threadIdx.x] = m2;
        __syncthreads();
        if (threadIdx.x >= L.slots) return;
        for (int q = 1; q < L.rpp; ++q)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                mean.e[k] += red[0][threadIdx.x + q * L.slots].e[k];
                m2.e[k] += red[1][threadIdx.x + q * L.slots].e[k];
            }
        const float inv = 1.0f / (float)(rows > 0 ? rows : 1);
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k >= L.skip) {
                p[k] = sh.e[k] + mean.e[k] * inv;             // a chunk without rows: zeros
                p[A.C + k] = fmaxf(m2.e[k] - mean.e[k] * mean.e[k] * inv, 0.f);
            }
        return;
    }
    if (rows > 0) {
        const VecF<V> a = ldv<T, V>(x + (L.r0 + rows / 5) * A.C), b = ldv<T, V>(x + (L.r0 + rows * 3 / 7) * A.C),
                      c = ldv<T, V>(x + (L.r0 + rows * 6 / 7) * A.C);
#pragma unroll
        for (int k = 0; k < V; ++k) sh.e[k] = __builtin_amdgcn_fmed3f(a.e[k], b.e[k], c.e[k]);
    }
    float n = 0.f;
    auto fold = [&](const VecF<V> &m, const VecF<V> &q, float rows) {
        const float all = n + rows, part = rows / all, both = n * part;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float d = m.e[k] - mean.e[k];
            mean.e[k] = fmaf(d, part, mean.e[k]);
            m2.e[k] += fmaf(d * d, both, q.e[k]);
        }
        n = all;
    };
    auto take = [&](long long r, int have) {        // `have` rows from r on, rpp apart
        VecF<V> v[kGnRows], m, q;
#pragma unroll
        for (int i = 0; i < kGnRows; ++i) v[i] = ldv<T, V>(x + (r + (i < have ? i : 0) * (long long)L.rpp) * A.C);
#pragma unroll
        for (int k = 0; k < V; ++k) m.e[k] = q.e[k] = 0.f;
        const float inv = 1.0f / (float)have;
#pragma unroll
        for (int i = 0; i < kGnRows; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[i].e[k] -= sh.e[k];
                m.e[k] += i < have ? v[i].e[k] : 0.f;
            }
#pragma unroll
        for (int k = 0; k < V; ++k) m.e[k] *= inv;
#pragma unroll
        for (int i = 0; i < kGnRows; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = v[i].e[k] - m.e[k];
                q.e[k] = i < have ? fmaf(d, d, q.e[k]) : q.e[k];
            }
        fold(m, q, (float)have);
    };
    if (L.on) {
        long long r = L.r0 + L.rsub;
        for (; r + (kGnRows - 1) * (long long)L.rpp < L.r1; r += kGnRows * (long long)L.rpp) take(r, kGnRows);
        if (r + 2ll * L.rpp < L.r1) {
            take(r, (int)((L.r1 - 1 - r) / L.rpp) + 1);
        } else {
            for (; r < L.r1; r += L.rpp) {                  // one or two
                VecF<V> v = ldv<T, V>(x + r * A.C), q;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    v.e[k] -= sh.e[k];
                    q.e[k] = 0.f;
                }
                fold(v, q, 1.f);
            }
        }
    }
    // the lanes of a channel by pairs
    for (int s = 1; s < L.rpp; s <<= 1) {
        red[0][threadIdx.x] = mean;
        red[1][threadIdx.x] = m2;
        count[threadIdx.x] = n;
        __syncthreads();
        if (L.on && L.rsub % (2 * s) == 0 && L.rsub + s < L.rpp) {
            const int at = threadIdx.x + s * L.slots;
            if (count[at] > 0.f) fold(red[0][at], red[1][at], count[at]);
        }
        __syncthreads();
    }
    if (threadIdx.x < L.slots) {
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k >= L.skip) {
                p[k] = sh.e[k] + mean.e[k];                  // a chunk without rows: zeros
                p[A.C + k] = m2.e[k];
            }
    }
}

// sum over a block's threads: waves first, then their sums in order
__device__ __forceinline__ double block_sum(double v, double *red) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0.0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) r += red[w];
    return r;
}

// Threads of a block over a [chunks][width] array: thread -> (channel, first chunk); a block takes `step`
// chunks at once, or several channels a thread when a group is wider than the block.
struct GnWalk {
    int j, c, step, jstep;
};
__device__ __forceinline__ GnWalk gn_walk(int width) {
    GnWalk w;
    const int lanes = width < (int)blockDim.x ? width : (int)blockDim.x;
    w.step = blockDim.x / lanes;
    w.j = threadIdx.x % lanes;
    w.c = threadIdx.x / lanes;
    w.jstep = lanes;
    if (w.c >= w.step) w.j = width;      // left over: nothing
    return w;
}

// one block per (group, sample): Chan over the group's channels and chunks, in double
__global__ __launch_bounds__(kGnJoin) void gn_finalize_kernel(const GnArgs A) {
    __shared__ double red[kGnJoin / 64];
    const int g = blockIdx.x;
    const int per = (int)((A.length + A.chunks - 1) / A.chunks);
    const int full = (int)(A.length / per), rest = (int)(A.length - (long long)full * per);
    const float *p = A.part + (long long)blockIdx.y * A.chunks * 2 * A.C + g * A.width;
    const GnWalk w = gn_walk(A.width);
    // deviations from one of the chunk means: what a difference of squares loses is then of the spread's size
    const float ref = p[0];
    double s = 0.0, q = 0.0;
    for (int j = w.j; j < A.width; j += w.jstep)
#pragma unroll 8
        for (int c = w.c; c < A.chunks; c += w.step) {
            const double rows = c < full ? per : (c == full ? rest : 0);
            const double d = (double)p[(long long)c * 2 * A.C + j] - ref;
            const double nd = rows > 0.0 ? rows * d : 0.0;
            s += nd;
            q += p[(long long)c * 2 * A.C + A.C + j] + nd * d;
        }
    const double count = (double)A.length * A.width;
    const double off = block_sum(s, red) / count, mean = ref + off;
    double var = block_sum(q, red) / count - off * off;
    var = var < 0.0 ? 0.0 : var;
    if (threadIdx.x == 0) {
        A.mean[(long long)blockIdx.y * A.groups + g] = (float)mean;
        A.rstd[(long long)blockIdx.y * A.groups + g] = (float)(1.0 / sqrt(var + (double)A.eps));
    }
}

// the lane's per-channel constants
template <class T, int V> struct GnCols {
    VecF<V> w, b, mean, rstd;
    __device__ __forceinline__ void load(const GnArgs &A, int off, long long sample) {
        w = ldv<T, V>(static_cast<const T *>(A.w) + off);
        b = ldv<T, V>(static_cast<const T *>(A.b) + off);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const long long g = sample * A.groups + (off + k) / A.width;
            mean.e[k] = A.mean[g];
            rstd.e[k] = A.rstd[g];
        }
    }
};

template <class T, int V, int ACT> __global__ __launch_bounds__(256) void gn_apply_fwd_kernel(const GnArgs A) {
    const GnLay L = gn_lay<V>(A);
    if (!L.on) return;
    const long long at = (long long)blockIdx.y * A.length * A.C + L.off;
    const T *x = static_cast<const T *>(A.x) + at;
    T *y = static_cast<T *>(A.y) + at;
    GnCols<T, V> P;
    P.load(A, L.off, blockIdx.y);
#pragma unroll 4
    for (long long r = L.r0 + L.rsub; r < L.r1; r += L.rpp) {
        VecF<V> v = ldv<T, V>(x + r * A.C);
#pragma unroll
        for (int k = 0; k < V; ++k)
            v.e[k] = act_value<ACT, IsF32<T>::value>(
                fmaf((v.e[k] - P.mean.e[k]) * P.rstd.e[k], P.w.e[k], P.b.e[k]));
        stv<T, V>(y + r * A.C, v);
    }
}

// per (sample, chunk, channel): sum du, sum du xh -> part
template <class T, int V, int ACT> __global__ __launch_bounds__(256) void gn_reduce_bwd_kernel(const GnArgs A) {
    __shared__ VecF<V> red[2][256];
    const GnLay L = gn_lay<V>(A);
    const long long at = (long long)blockIdx.y * A.length * A.C + L.off;
    const T *x = static_cast<const T *>(A.x) + at, *dy = static_cast<const T *>(A.dy) + at;
    VecF<V> s1, s2;
#pragma unroll
    for (int k = 0; k < V; ++k) s1.e[k] = s2.e[k] = 0.f;
    if (L.on) {
        GnCols<T, V> P;
        P.load(A, L.off, blockIdx.y);
#pragma unroll 2
        for (long long r = L.r0 + L.rsub; r < L.r1; r += L.rpp) {
            const VecF<V> v = ldv<T, V>(x + r * A.C), g = ldv<T, V>(dy + r * A.C);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float xh = (v.e[k] - P.mean.e[k]) * P.rstd.e[k];
                float d;
                act_both<ACT, IsF32<T>::value>(fmaf(xh, P.w.e[k], P.b.e[k]), d);
                const float du = g.e[k] * d;
                s1.e[k] += du;
                s2.e[k] = fmaf(du, xh, s2.e[k]);
            }
        }
    }
    red[0][threadIdx.x] = s1;
    red[1][threadIdx.x] = s2;
    __syncthreads();
    if (threadIdx.x < L.slots) {
        for (int q = 1; q < L.rpp; ++q)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                s1.e[k] += red[0][threadIdx.x + q * L.slots].e[k];
                s2.e[k] += red[1][threadIdx.x + q * L.slots].e[k];
            }
        float *p = A.part + ((long long)blockIdx.y * A.chunks + blockIdx.x) * 2 * A.C + L.off;
#pragma unroll
        for (int k = 0; k < V; ++k)
            if (k >= L.skip) {
                p[k] = s1.e[k];
                p[A.C + k] = s2.e[k];
            }
    }
}

// one block per (group, sample): mean(g) and mean(g xh) of the group
template <class T> __global__ __launch_bounds__(kGnJoin) void gn_coef_kernel(const GnArgs A) {
    __shared__ double red[kGnJoin / 64];
    const int g = blockIdx.x;
    const float *p = A.part + (long long)blockIdx.y * A.chunks * 2 * A.C + g * A.width;
    const T *w = static_cast<const T *>(A.w) + g * A.width;
    const GnWalk k = gn_walk(A.width);
    double s1 = 0.0, s2 = 0.0;
    for (int j = k.j; j < A.width; j += k.jstep) {
        const double wj = (float)w[j];
#pragma unroll 8
        for (int c = k.c; c < A.chunks; c += k.step) {
            s1 += wj * p[(long long)c * 2 * A.C + j];
            s2 += wj * p[(long long)c * 2 * A.C + A.C + j];
        }
    }
    const double count = (double)A.length * A.width;
    const double m1 = block_sum(s1, red) / count, m2 = block_sum(s2, red) / count;
    if (threadIdx.x == 0) {
        float *o = A.coef + ((long long)blockIdx.y * A.groups + g) * 2;
        o[0] = (float)m1;
        o[1] = (float)m2;
    }
}

template <class T, int V, int ACT> __global__ __launch_bounds__(256) void gn_apply_bwd_kernel(const GnArgs A) {
    const GnLay L = gn_lay<V>(A);
    if (!L.on) return;
    const long long at = (long long)blockIdx.y * A.length * A.C + L.off;
    const T *x = static_cast<const T *>(A.x) + at, *dy = static_cast<const T *>(A.dy) + at;
    T *dx = static_cast<T *>(A.dx) + at;
    GnCols<T, V> P;
    P.load(A, L.off, blockIdx.y);
    VecF<V> m1, m2;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const float *o = A.coef + ((long long)blockIdx.y * A.groups + (L.off + k) / A.width) * 2;
        m1.e[k] = o[0];
        m2.e[k] = o[1];
    }
#pragma unroll 4
    for (long long r = L.r0 + L.rsub; r < L.r1; r += L.rpp) {
        const VecF<V> v = ldv<T, V>(x + r * A.C);
        VecF<V> g = ldv<T, V>(dy + r * A.C);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float xh = (v.e[k] - P.mean.e[k]) * P.rstd.e[k];
            float d;
            act_both<ACT, IsF32<T>::value>(fmaf(xh, P.w.e[k], P.b.e[k]), d);
            g.e[k] = P.rstd.e[k] * (g.e[k] * d * P.w.e[k] - m1.e[k] - xh * m2.e[k]);
        }
        stv<T, V>(dx + r * A.C, g);
    }
}

// ---- column sums of f32 partials, in two fixed-order steps -------------------------------------
// slab[s][k][c] = sum over this slab's rows of in[k][row][c];  then out_k[c] = sum over slabs.
// Row `r` of column set k starts at in + k * set + r * ld.
__global__ __launch_bounds__(256) void colsum_slab_kernel(const float *in, long long rows, long long ld,
                                                          long long set, int cols, float *slab) {
    __shared__ float red[256];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), rg = threadIdx.x >> 5;
    const long long per = (rows + gridDim.y - 1) / gridDim.y;
    const long long r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    float s = 0.f;
    if (c < cols)
#pragma unroll 8
        for (long long r = r0 + rg; r < r1; r += 8) s += in[blockIdx.z * set + r * ld + c];
    red[threadIdx.x] = s;
    __syncthreads();
    if (rg == 0 && c < cols) {
        for (int q = 1; q < 8; ++q) s += red[threadIdx.x + q * 32];
        slab[((long long)blockIdx.y * gridDim.z + blockIdx.z) * cols + c] = s;
    }
}
// (few rows: the rows themselves as slabs)
template <class T>
__global__ __launch_bounds__(256) void colsum_final_kernel(const float *slab, int nslab, long long ld, long long set,
                                                           int cols, T *out0, T *out1) {
    __shared__ double red[256];
    const int i = blockIdx.x * 32 + (threadIdx.x & 31), rg = threadIdx.x >> 5;     // i over [2][cols]
    const float *at = i < cols ? slab + i : slab + set + (i - cols);
    double s = 0.0;
    if (i < 2 * cols)
#pragma unroll 8
        for (int q = rg; q < nslab; q += 8) s += at[q * ld];
    red[threadIdx.x] = s;
    __syncthreads();
    if (rg == 0 && i < 2 * cols) {
        for (int q = 1; q < 8; ++q) s += red[threadIdx.x + q * 32];
        T *o = i < cols ? out0 + i : out1 + (i - cols);
        *o = (T)(float)s;
    }
}

// a group that fits the registers of one wave and is contiguous
static bool gn_in_registers(const gatmi_group_norm *g) {
    return g->length == 1 && g->width <= 64 * (g->dtype == GATMI_F32 ? 4 : 8) * kGnMaxT;
}

static int gn_check(const gatmi_group_norm *g) {
    GATMI_REQUIRE(g, "null group norm descriptor");
    GATMI_REQUIRE(g->dtype >= GATMI_F32 && g->dtype <= GATMI_F16, "group_norm: unknown element type %d", g->dtype);
    GATMI_REQUIRE(g->act >= GATMI_ACT_NONE && g->act <= GATMI_ACT_GELU, "group_norm: unknown activation %d", g->act);
    GATMI_REQUIRE(g->groups >= 1 && g->width >= 1 && (long long)g->groups * g->width <= GATMI_GROUP_NORM_MAX_CHANNELS,
                  "group_norm: %d groups of %d channels (at most %d channels in all)", g->groups, g->width,
                  GATMI_GROUP_NORM_MAX_CHANNELS);
    GATMI_REQUIRE(g->batch >= 0 && g->length >= 1 && g->batch < (1ll << 31) && g->length < (1ll << 31),
                  "group_norm: batch %lld / length %lld out of range", (long long)g->batch, (long long)g->length);
    GATMI_REQUIRE(g->eps >= 0.f, "group_norm: negative eps");
    return GATMI_OK;
}

struct GnGeom {
    bool seg;       // the segment form
    int V, TT, W, w_log;
    int blocks_fwd, blocks_bwd;
    long long slots;      // lane groups of the backward's grid
    int chunks, apply, zblocks;      // row ranges a sample is cut into
    int join;             // threads of a joining block
    int slabs;
    size_t part_floats, slab_floats, coef_floats;
};

static int igcd(int a, int b) { return b ? igcd(b, a % b) : a; }

static GnGeom gn_geom(const gatmi_group_norm *g) {
    GnGeom G;
    memset(&G, 0, sizeof(G));
    const int C = g->groups * g->width;
    G.seg = gn_in_registers(g);
    if (G.seg) {
        G.V = vec_of(g->dtype, g->width);
        const int nv = (g->width + G.V - 1) / G.V;
        G.W = nv >= 64 ? 64 : next_pow2(nv);
        G.w_log = ilog2(G.W);
        G.TT = next_pow2((nv + G.W - 1) / G.W);
        const int per_block = 256 >> G.w_log;
        const int unit = g->groups / igcd(g->groups, per_block);   // blocks whose segments are whole samples
        const long long nseg = g->batch * (long long)g->groups;
        const long long need = (nseg + per_block - 1) / per_block;
        auto grid = [&](long long most) {
            long long b = need < most ? need : most;
            b = (b + unit - 1) / unit * unit;
            return (int)(b < unit ? unit : b);
        };
        G.blocks_fwd = grid(kGnFwdBlocks);
        G.blocks_bwd = grid(kGnBwdBlocks);
        G.slots = (long long)G.blocks_bwd * per_block;
        G.part_floats = (size_t)2 * G.slots * g->width;
    } else {
        G.V = vec_of(g->dtype, C);
        const int nslot = (C + G.V - 1) / G.V;
        G.zblocks = (nslot + 255) / 256;
        const int rpp = nslot < 256 ? 256 / nslot : 1;
        // at least eight rows a lane; at most kGnChunks blocks over all samples
        const long long want = (g->length + 8ll * rpp - 1) / (8ll * rpp);
        const long long lots = (long long)G.zblocks * (g->batch > 0 ? g->batch : 1);
        auto cut = [&](long long blocks) {
            const long long most = blocks / lots < 1 ? 1 : blocks / lots;
            return (int)(want < most ? want : most);
        };
        G.chunks = cut(kGnChunks);
        G.apply = cut(kGnApply);
        // about four values a thread: many samples of a few chunks each take a wave per group, not sixteen
        G.join = next_pow2(G.chunks * g->width / 4 + 1);
        G.join = G.join < 64 ? 64 : (G.join > kGnJoin ? kGnJoin : G.join);
        G.part_floats = (size_t)g->batch * G.chunks * 2 * C;
        G.coef_floats = (size_t)g->batch * g->groups * 2;
    }
    G.slabs = kGnSlabs;
    G.slab_floats = (size_t)G.slabs * 2 * C;
    return G;
}

static void gn_fill(GnArgs &A, const gatmi_group_norm *g, const GnGeom &G) {
    memset(&A, 0, sizeof(A));
    A.w = g->weight;
    A.b = g->bias;
    A.nseg = g->batch * (long long)g->groups;
    A.length = g->length;
    A.groups = g->groups;
    A.width = g->width;
    A.C = g->groups * g->width;
    A.chunks = G.chunks;
    A.W = G.W;
    A.w_log = G.w_log;
    A.eps = g->eps;
    A.inv_n = 1.0f / (float)g->width;
}

// f(samples, their arguments) of the chunk form: a launch takes at most kGnSamples samples (grid.y)
template <class F> static void gn_slices(const gatmi_group_norm *g, const GnArgs &all, F f) {
    const long long el = g->dtype == GATMI_F32 ? 4 : 2, sample = g->length * all.C * el;
    auto move = [](auto *&p, long long bytes) {
        if (p) p = reinterpret_cast<std::remove_reference_t<decltype(p)>>((uintptr_t)p + bytes);
    };
    for (long long s = 0; s < g->batch; s += kGnSamples) {
        GnArgs A = all;
        move(A.x, s * sample);
        move(A.dy, s * sample);
        move(A.y, s * sample);
        move(A.dx, s * sample);
        A.mean += s * A.groups;
        A.rstd += s * A.groups;
        A.part += s * A.chunks * 2 * A.C;
        if (A.coef) A.coef += s * A.groups * 2;
        f((unsigned)(g->batch - s < kGnSamples ? g->batch - s : kGnSamples), A);
    }
}

// f(V, TT) of the segment form: several vectors a lane only when they are full ones
template <class T, class F> static void with_seg(const GnGeom &G, F f) {
    with_vec<T>(G.V, [&](auto V) {
        if constexpr (decltype(V)::value == 16 / sizeof(T)) {
            if (G.TT == 2) return f(V, std::integral_constant<int, 2>{});
            if (G.TT == 4) return f(V, std::integral_constant<int, 4>{});
            if (G.TT == 8) return f(V, std::integral_constant<int, 8>{});
        }
        f(V, std::integral_constant<int, 1>{});
    });
}

}  // namespace gatmi

using namespace gatmi;

extern "C" size_t gatmi_group_norm_workspace_bytes(const gatmi_group_norm *g) {
    if (gn_check(g)) return 0;
    const GnGeom G = gn_geom(g);
    return align_up(G.part_floats * 4) + align_up(G.slab_floats * 4) + align_up(G.coef_floats * 4) + 256;
}

extern "C" int gatmi_group_norm_fwd(const gatmi_group_norm *g, const void *x, void *y, float *mean, float *rstd,
                                    void *ws, size_t ws_bytes, void *stream) {
    if (int e = gn_check(g)) return e;
    if (g->batch == 0) return GATMI_OK;
    GATMI_REQUIRE(x && y && g->weight && g->bias, "group_norm_fwd: null argument");
    GATMI_REQUIRE(!mean == !rstd, "group_norm_fwd: mean and rstd are saved together or not at all");
    const GnGeom G = gn_geom(g);
    hipStream_t st = static_cast<hipStream_t>(stream);
    GnArgs A;
    gn_fill(A, g, G);
    A.x = x;
    A.y = y;
    A.mean = mean;
    A.rstd = rstd;
    if (G.seg) {
        ProfScope ps("group_norm_seg_fwd", st);
        GATMI_WITH_TYPE(g->dtype, GATMI_WITH_ACT(g->act, with_seg<T>(G, [&](auto V, auto TT) {
            constexpr int v = decltype(V)::value, t = decltype(TT)::value;
            if (mean) hipLaunchKernelGGL((gn_seg_fwd_kernel<T, v, t, ACT, true>), dim3(G.blocks_fwd), dim3(256), 0, st, A);
            else hipLaunchKernelGGL((gn_seg_fwd_kernel<T, v, t, ACT, false>), dim3(G.blocks_fwd), dim3(256), 0, st, A);
        })));
        GATMI_HIP(hipGetLastError());
        return GATMI_OK;
    }
    GATMI_REQUIRE(mean, "group_norm_fwd: this shape needs mean and rstd");
    if (ws_bytes < gatmi_group_norm_workspace_bytes(g) || !ws) {
        set_error("group_norm workspace too small: %zu < %zu", ws_bytes, gatmi_group_norm_workspace_bytes(g));
        return GATMI_ERR_WS;
    }
    A.part = static_cast<float *>(ws);
    ProfScope ps("group_norm_fwd", st);
    gn_slices(g, A, [&](unsigned samples, GnArgs S) {
        const dim3 grid(G.chunks, samples, G.zblocks), apply(G.apply, samples, G.zblocks);
        const bool few = (g->length + G.chunks - 1) / G.chunks <= kGnFew;
        GATMI_WITH_TYPE(g->dtype, with_vec<T>(G.V, [&](auto V) {
            if (few) hipLaunchKernelGGL((gn_stats_kernel<T, decltype(V)::value, true>), grid, dim3(256), 0, st, S);
            else hipLaunchKernelGGL((gn_stats_kernel<T, decltype(V)::value, false>), grid, dim3(256), 0, st, S);
        }));
        hipLaunchKernelGGL(gn_finalize_kernel, dim3(g->groups, samples), dim3(G.join), 0, st, S);
        S.chunks = G.apply;
        GATMI_WITH_TYPE(g->dtype, GATMI_WITH_ACT(g->act, with_vec<T>(G.V, [&](auto V) {
            hipLaunchKernelGGL((gn_apply_fwd_kernel<T, decltype(V)::value, ACT>), apply, dim3(256), 0, st, S);
        })));
    });
    GATMI_HIP(hipGetLastError());
    return GATMI_OK;
}

extern "C" int gatmi_group_norm_bwd(const gatmi_group_norm *g, const void *x, const void *grad_y, const float *mean,
                                    const float *rstd, void *grad_x, void *grad_weight, void *grad_bias, void *ws,
                                    size_t ws_bytes, void *stream) {
    if (int e = gn_check(g)) return e;
    GATMI_REQUIRE(grad_weight && grad_bias && g->weight && g->bias, "group_norm_bwd: null argument");
    GATMI_REQUIRE(g->batch == 0 || (x && grad_y && mean && rstd && grad_x), "group_norm_bwd: null argument");
    if (ws_bytes < gatmi_group_norm_workspace_bytes(g) || !ws) {
        set_error("group_norm workspace too small: %zu < %zu", ws_bytes, gatmi_group_norm_workspace_bytes(g));
        return GATMI_ERR_WS;
    }
    const GnGeom G = gn_geom(g);
    hipStream_t st = static_cast<hipStream_t>(stream);
    GnArgs A;
    gn_fill(A, g, G);
    A.x = x;
    A.dy = grad_y;
    A.dx = grad_x;
    A.mean = const_cast<float *>(mean);
    A.rstd = const_cast<float *>(rstd);
    Carver cv(ws);
    A.part = cv.take<float>(G.part_floats);
    float *slab = cv.take<float>(G.slab_floats);
    A.coef = cv.take<float>(G.coef_floats);
    const int C = A.C;
    long long rows = 0, ld = 0, set = 0;     // of the partial sums: (dw, db)
    void *out0 = grad_weight, *out1 = grad_bias;
    if (g->batch > 0 && G.seg) {
        ProfScope ps("group_norm_seg_bwd", st);
        GATMI_WITH_TYPE(g->dtype, GATMI_WITH_ACT(g->act, with_seg<T>(G, [&](auto V, auto TT) {
            hipLaunchKernelGGL((gn_seg_bwd_kernel<T, decltype(V)::value, decltype(TT)::value, ACT>), dim3(G.blocks_bwd),
                               dim3(256), 0, st, A);
        })));
        GATMI_HIP(hipGetLastError());
        rows = G.slots / g->groups;          // slot k * groups + j -> row k, channels of group j
        ld = C;
        set = G.slots * (long long)g->width;
    } else if (g->batch > 0) {
        ProfScope ps("group_norm_bwd", st);
        gn_slices(g, A, [&](unsigned samples, GnArgs S) {
            const dim3 grid(G.chunks, samples, G.zblocks), apply(G.apply, samples, G.zblocks);
            GATMI_WITH_TYPE(g->dtype, GATMI_WITH_ACT(g->act, with_vec<T>(G.V, [&](auto V) {
                hipLaunchKernelGGL((gn_reduce_bwd_kernel<T, decltype(V)::value, ACT>), grid, dim3(256), 0, st, S);
            })));
            GATMI_WITH_TYPE(g->dtype, hipLaunchKernelGGL((gn_coef_kernel<T>), dim3(g->groups, samples), dim3(G.join), 0,
                                                         st, S));
            S.chunks = G.apply;
            GATMI_WITH_TYPE(g->dtype, GATMI_WITH_ACT(g->act, with_vec<T>(G.V, [&](auto V) {
                hipLaunchKernelGGL((gn_apply_bwd_kernel<T, decltype(V)::value, ACT>), apply, dim3(256), 0, st, S);
            })));
        });
        GATMI_HIP(hipGetLastError());
        rows = g->batch * G.chunks;
        ld = 2ll * C;
        set = C;                             // row: [sum du][sum du xh]
        out0 = grad_bias;
        out1 = grad_weight;
    }
    ProfScope ps("group_norm_param_sums", st);
    const float *sums = A.part;
    int nsum = (int)rows;
    if (rows > 4 * G.slabs) {
        hipLaunchKernelGGL(colsum_slab_kernel, dim3((C + 31) / 32, G.slabs, 2), dim3(256), 0, st, A.part, rows, ld, set,
                           C, slab);
        sums = slab;
        nsum = G.slabs;
        ld = 2ll * C;
        set = C;
    }
    GATMI_WITH_TYPE(g->dtype, hipLaunchKernelGGL((colsum_final_kernel<T>), dim3((2 * C + 31) / 32), dim3(256), 0, st,
                                                 sums, nsum, ld, set, C, static_cast<T *>(out0),
                                                 static_cast<T *>(out1)));
    GATMI_HIP(hipGetLastError());
    return GATMI_OK;
}
