// Embedding lookup with scaling, and its gradient by sorted ids.
//   forward   y[i, :] = scale * table[ids[i], :]            (a zero row where ids[i] is outside [0, vocab))
//   backward  dtable[v, :] = scale * sum_{i : ids[i] = v} dy[i, :]
//
// The gradient is a segmented sum: a stable radix sort of (id, position) puts the rows of one table entry
// side by side, in the order of the positions, and the sorted list is summed in fixed chunks of rows -- so
// that one frequent id costs what many rare ones do -- whose unfinished ends are summed the same way, level
// by level.  No float atomics: the order of every sum is fixed by the ids alone.
//
// 2449029 ids of [1000003, 128] bf16: forward 189 us (627 MB written, the table's rows mostly from the caches),
// backward 390: 40 to clear the table (256 MB, 6.4 TB/s), 120 for three passes of the sort, 197 for the sum
// (627 MB of dy read in random order of its rows), 42 for the ends.  200000 ids of [65536, 30] f32: 8.5 us forward;
// the backward's 70 us are ten dependent launches of 3 to 15 us each.
#include "attn_device.h"
#include "common.h"
#include "dense_device.h"

namespace gatmi {

// ---- forward ---------------------------------------------------------------------------------
constexpr int kEmbUnroll = 4;

struct EmbArgs {
    const int64_t *ids;
    const void *table;
    void *y;
    long long n, vocab;
    int dim, W, w_log;     // W lanes a row
    float scale;
};

template <class T, int V> __global__ __launch_bounds__(256) void emb_fwd_kernel(const EmbArgs A) {
    const int lane = threadIdx.x & (A.W - 1);
    const int per_block = 256 >> A.w_log;
    const T *table = static_cast<const T *>(A.table);
    T *y = static_cast<T *>(A.y);
    const long long first = (long long)blockIdx.x * (per_block * kEmbUnroll) + (threadIdx.x >> A.w_log);
    long long id[kEmbUnroll];
#pragma unroll
    for (int u = 0; u < kEmbUnroll; ++u) {
        const long long i = first + u * per_block;
        id[u] = i < A.n ? A.ids[i] : -1;
    }
    for (int j0 = lane * V; j0 < A.dim; j0 += A.W * V) {
        const int j = j0 + V <= A.dim ? j0 : A.dim - V;     // the last vector steps back (equal stores)
        VecF<V> v[kEmbUnroll];
#pragma unroll
        for (int u = 0; u < kEmbUnroll; ++u) {
            if (id[u] >= 0 && id[u] < A.vocab) {
                v[u] = ldv<T, V>(table + id[u] * A.dim + j);
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k) v[u].e[k] = 0.f;
            }
        }
#pragma unroll
        for (int u = 0; u < kEmbUnroll; ++u) {
            const long long i = first + u * per_block;
            if (i >= A.n) continue;
#pragma unroll
            for (int k = 0; k < V; ++k) v[u].e[k] *= A.scale;
            stv<T, V>(y + i * A.dim + j, v[u]);
        }
    }
}

// ---- gradient --------------------------------------------------------------------------------
// `bytes` at p set to zero, by `blocks` blocks of which this is number `b`: the aligned middle in 16-byte
// stores, the few bytes around it one by one
__device__ __forceinline__ void zero_fill(char *p, long long bytes, int b, int blocks) {
    const long long lead = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15, head = lead < bytes ? lead : bytes;
    const long long n16 = (bytes - head) / 16, rest = bytes - head - n16 * 16;
    uint4 *q = reinterpret_cast<uint4 *>(p + head);
    for (long long i = b * 256ll + threadIdx.x; i < n16; i += blocks * 256ll) q[i] = make_uint4(0, 0, 0, 0);
    if (b == 0 && threadIdx.x < 16) {
        if ((long long)threadIdx.x < head) p[threadIdx.x] = 0;
        if ((long long)threadIdx.x < rest) p[head + n16 * 16 + threadIdx.x] = 0;
    }
}

// ---- stable radix sort of (id, position) ---------------------------------------------------------
// `bits` (at most 9) of the key a pass: with more, a tile's runs of equal digits get shorter than a cache
// line and the scattered stores cost more than the pass saved.  A block owns a
// tile of 256 * ITEMS consecutive items; wave w of it the items [w * 64 * ITEMS, ..), 64 at a time: an
// item's rank is what came before it in (tile, wave, step, lane) order, which is the order of the items.
constexpr int kSortMaxBits = 9, kSmallSort = 4096;

struct SortArgs {
    const int64_t *ids;            // first pass: keys come from here, positions are the indices
    const uint2 *in;               // later ones: (key, position)
    uint2 *out;
    uint32_t *hist;                // [bins][blocks]
    uint32_t *total;               // [bins]
    long long n, vocab;
    int blocks, shift, bits, passes;
};

// ids outside the table get the key `vocab`: they sort behind every row and are left out of the sums
__device__ __forceinline__ uint32_t id_key(int64_t id, long long vocab) {
    return (uint32_t)(id >= 0 && id < vocab ? id : vocab);
}
__device__ __forceinline__ uint32_t sort_key(const SortArgs &A, long long i) {
    return A.ids ? id_key(A.ids[i], A.vocab) : A.in[i].x;
}

// Lanes of this wave whose digit equals this lane's (only lanes with `on` count)
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool on) {
    uint64_t m = __ballot(on);
    for (int b = 0; b < bits; ++b) {
        const uint64_t bit = __ballot((digit >> b) & 1u);
        m &= (digit >> b) & 1u ? bit : ~bit;
    }
    return m;
}

// Ranks this wave's items among the wave's equal digits: rank[k], and the wave's counts in `cnt` [bins],
// zero before.  volatile: lanes read each other's counts; a wave's LDS accesses are in order.
template <int ITEMS>
__device__ __forceinline__ void wave_ranks(volatile uint32_t *cnt, const uint32_t (&digit)[ITEMS], int have, int bits,
                                           int lane, uint32_t (&rank)[ITEMS]) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const bool on = k * 64 + lane < have;
        const uint64_t m = same_digit(digit[k], bits, on);
        const uint32_t before = __popcll(m & ((1ull << lane) - 1ull));
        const uint32_t seen = on ? cnt[digit[k]] : 0u;
        rank[k] = seen + before;
        if (on && before == 0) cnt[digit[k]] = seen + (uint32_t)__popcll(m);
        __builtin_amdgcn_wave_barrier();
    }
}

// Exclusive scan over the block's 256 threads
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *wsum, uint32_t *all = nullptr) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(s, o, 64);
        if (lane >= o) s += up;
    }
    if (lane == 63) wsum[wave] = s;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += wsum[w];
    if (all) *all = wsum[0] + wsum[1] + wsum[2] + wsum[3];
    __syncthreads();
    return before + s - v;
}

template <int ITEMS> __global__ __launch_bounds__(256) void sort_count_kernel(const SortArgs A) {
    extern __shared__ uint32_t h[];
    const int bins = 1 << A.bits;
    for (int d = threadIdx.x; d < bins; d += 256) h[d] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * (256 * ITEMS);
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const long long i = base + k * 256 + threadIdx.x;
        if (i < A.n) atomicAdd(&h[(sort_key(A, i) >> A.shift) & (bins - 1)], 1u);   // integers: any order
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += 256) A.hist[(long long)d * A.blocks + blockIdx.x] = h[d];
}

// block d: exclusive scan of digit d's counts over the tiles; total[d]
__global__ __launch_bounds__(256) void sort_scan_kernel(const SortArgs A) {
    __shared__ uint32_t wsum[4];
    uint32_t *row = A.hist + (long long)blockIdx.x * A.blocks;
    uint32_t carry = 0;
    for (int base = 0; base < A.blocks; base += 256) {
        const int i = base + threadIdx.x;
        const uint32_t v = i < A.blocks ? row[i] : 0;
        uint32_t all;
        const uint32_t before = block_scan(v, wsum, &all);
        if (i < A.blocks) row[i] = carry + before;
        carry += all;
    }
    if (threadIdx.x == 0) A.total[blockIdx.x] = carry;
}

template <int ITEMS> __global__ __launch_bounds__(256) void sort_scatter_kernel(const SortArgs A) {
    extern __shared__ uint32_t smem[];
    __shared__ uint32_t wsum[4];
    volatile uint32_t *cnt = smem;       // [4][bins]
    const int bins = 1 << A.bits;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = threadIdx.x; d < 4 * bins; d += 256) cnt[d] = 0;
    __syncthreads();
    const long long base = (long long)blockIdx.x * (256 * ITEMS) + wave * (64 * ITEMS);
    const long long left = A.n - base;
    const int have = left < 0 ? 0 : (left < 64 * ITEMS ? (int)left : 64 * ITEMS);
    uint32_t key[ITEMS], pos[ITEMS], digit[ITEMS], rank[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const long long i = base + k * 64 + lane;
        const bool on = k * 64 + lane < have;
        uint2 e = make_uint2(0u, 0u);
        if (on) e = A.ids ? make_uint2(id_key(A.ids[i], A.vocab), (uint32_t)i) : A.in[i];
        key[k] = e.x;
        pos[k] = e.y;
        digit[k] = (key[k] >> A.shift) & (bins - 1);
    }
    // this thread's digits, at most two: their counts are on their way while the wave ranks its items
    constexpr int kDigits = (1 << kSortMaxBits) / 256;
    const int per = bins > 256 ? kDigits : 1, d0 = threadIdx.x * per;
    uint32_t total[kDigits], before[kDigits];
#pragma unroll
    for (int q = 0; q < kDigits; ++q) {
        const bool on = q < per && d0 + q < bins;
        total[q] = on ? A.total[d0 + q] : 0u;
        before[q] = on ? A.hist[(long long)(d0 + q) * A.blocks + blockIdx.x] : 0u;
    }
    wave_ranks<ITEMS>(cnt + wave * bins, digit, have, A.bits, lane, rank);
    __syncthreads();
    // the tile's own order first, in LDS: neighbours in it go to neighbouring places, and the stores of a wave
    // become runs instead of 64 separate ones
    uint2 *tile = reinterpret_cast<uint2 *>(smem + 5 * bins);
    uint32_t *shift = smem + 4 * bins;       // [bins]: a digit's place in the output less its place in the tile
    {
        uint32_t mine = 0, all = 0;
#pragma unroll
        for (int q = 0; q < kDigits; ++q)
            if (q < per && d0 + q < bins) {
                for (int w = 0; w < 4; ++w) mine += cnt[w * bins + d0 + q];
                all += total[q];
            }
        uint32_t here = block_scan(mine, wsum), there = block_scan(all, wsum);
#pragma unroll
        for (int q = 0; q < kDigits; ++q) {
            const int d = d0 + q;
            if (q >= per || d >= bins) break;
            shift[d] = there + before[q] - here;
            there += total[q];
            for (int w = 0; w < 4; ++w) {
                const uint32_t c = cnt[w * bins + d];
                cnt[w * bins + d] = here;
                here += c;
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (k * 64 + lane < have) tile[cnt[wave * bins + digit[k]] + rank[k]] = make_uint2(key[k], pos[k]);
    __syncthreads();
    const long long first = (long long)blockIdx.x * (256 * ITEMS);
    const int n = A.n - first < 256 * ITEMS ? (int)(A.n - first) : 256 * ITEMS;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 256) {
        const uint2 e = tile[i];
        A.out[i + shift[(e.x >> A.shift) & (bins - 1)]] = e;
    }
}

// at most kSmallSort items: all passes in one block, through LDS.  The grid's other blocks clear the gradient.
__global__ __launch_bounds__(256) void sort_small_kernel(const SortArgs A, char *clear, long long bytes) {
    if (blockIdx.x > 0) {
        zero_fill(clear, bytes, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    constexpr int ITEMS = kSmallSort / 256;
    __shared__ uint32_t skey[kSmallSort], spos[kSmallSort], scnt[4 * 256], wsum[4];
    volatile uint32_t *cnt = scnt;
    constexpr int bins = 256;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = (int)A.n;
    const int base = wave * (64 * ITEMS);
    const int have = n - base < 0 ? 0 : (n - base < 64 * ITEMS ? n - base : 64 * ITEMS);
    uint32_t key[ITEMS], pos[ITEMS], digit[ITEMS], rank[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = base + k * 64 + lane;
        const bool on = k * 64 + lane < have;
        key[k] = on ? id_key(A.ids[i], A.vocab) : 0u;
        pos[k] = (uint32_t)i;
    }
    for (int p = 0; p < A.passes; ++p) {
        for (int d = threadIdx.x; d < 4 * bins; d += 256) cnt[d] = 0;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) digit[k] = (key[k] >> (8 * p)) & (bins - 1);
        __syncthreads();
        wave_ranks<ITEMS>(cnt + wave * bins, digit, have, 8, lane, rank);
        __syncthreads();
        uint32_t mine = 0;      // thread d: digit d
        for (int w = 0; w < 4; ++w) mine += cnt[w * bins + threadIdx.x];
        uint32_t at = block_scan(mine, wsum);
        for (int w = 0; w < 4; ++w) {
            const uint32_t c = cnt[w * bins + threadIdx.x];
            cnt[w * bins + threadIdx.x] = at;
            at += c;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
            if (k * 64 + lane < have) {
                const uint32_t to = cnt[wave * bins + digit[k]] + rank[k];
                skey[to] = key[k];
                spos[to] = pos[k];
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k)
            if (k * 64 + lane < have) {
                key[k] = skey[base + k * 64 + lane];
                pos[k] = spos[base + k * 64 + lane];
            }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k)
        if (k * 64 + lane < have) {
            A.out[base + k * 64 + lane] = make_uint2(key[k], pos[k]);
        }
}

// ---- segmented sum of the sorted rows -----------------------------------------------------------
// One level: entries [0, n) in order, equal keys side by side; entry e stands for row `row(e)` of the
// source (none: a key that only continues its neighbours).  A lane group walks a chunk of entries and
// stores every segment that lies inside the chunk; the parts of segments that cross its ends go to
// (first, last) entries of the next level.
constexpr uint32_t kNoKey = 0xffffffffu;

struct SegArgs {
    const uint2 *entry;           // (key, position) at level 0; above (key, 1 where the entry carries a row)
    const void *src;              // level 0: dy; level > 0: f32 partial rows
    void *out;                    // dtable
    uint2 *nentry;                // next level's entries, two a chunk
    float *nsrc;
    long long n;
    uint32_t vocab;
    int dim, chunk, W, w_log;
    int own_entries;              // every block of columns writes the entries (to a place of its own)
    float scale;
};

template <class T, class S, int V, bool LEAF>
__device__ __forceinline__ void seg_chunk(const SegArgs &A, long long c, int lane) {
    const long long e0 = c * A.chunk;
    const long long e1 = e0 + A.chunk < A.n ? e0 + A.chunk : A.n;
    const int j0 = (blockIdx.y * A.W + lane) * V;
    const bool on = j0 < A.dim;
    const int j = !on ? 0 : (j0 + V <= A.dim ? j0 : A.dim - V);
    const S *src = static_cast<const S *>(A.src) + j;
    T *out = static_cast<T *>(A.out) + j;
    const uint32_t before = e0 > 0 ? A.entry[e0 - 1].x : kNoKey, after = e1 < A.n ? A.entry[e1].x : kNoKey;
    const uint32_t head = A.entry[e0].x, tail = A.entry[e1 - 1].x;
    const bool open_head = head < A.vocab && head == before;
    const bool open_tail = tail < A.vocab && tail == after;
    uint32_t k0 = kNoKey, k1 = kNoKey, f0 = 0, f1 = 0;
    VecF<V> acc;
#pragma unroll
    for (int k = 0; k < V; ++k) acc.e[k] = 0.f;
    uint32_t cur = head;
    bool first = true;      // the chunk's first segment
    // Every entry names a row that exists, so rows are loaded without a test (past the end: the last entry
    // again) and the keys and positions of the next batch travel while this one's rows do.
    constexpr int U = 8;
    uint32_t kk[U], pp[U], kn[U], pn[U];
    auto entries = [&](long long e, uint32_t (&k_)[U], uint32_t (&p_)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long i = e + u < e1 ? e + u : e1 - 1;
            const uint2 en = A.entry[i];
            k_[u] = en.x;
            p_[u] = en.y;
        }
    };
    entries(e0, kn, pn);
    for (long long e = e0; e < e1; e += U) {
        VecF<V> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            kk[u] = kn[u];
            pp[u] = pn[u];
            const long long r = LEAF ? (long long)pp[u] : (e + u < e1 ? e + u : e1 - 1);
            v[u] = ldv<S, V>(src + r * A.dim);
        }
        entries(e + U, kn, pn);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (e + u >= e1) break;
            if (kk[u] != cur) {       // `cur` ends inside this chunk
                if (cur < A.vocab) {
                    if (first && open_head) {
                        k0 = cur;
                        f0 = 1;
                        if (on) stv<float, V>(A.nsrc + (2 * c) * A.dim + j, acc);
                    } else if (on) {
#pragma unroll
                        for (int k = 0; k < V; ++k) acc.e[k] *= A.scale;
                        stv<T, V>(out + (long long)cur * A.dim, acc);
                    }
                }
                first = false;
                cur = kk[u];
#pragma unroll
                for (int k = 0; k < V; ++k) acc.e[k] = 0.f;
            }
            if (LEAF || pp[u])        // a node entry without a row holds nothing that was written
#pragma unroll
                for (int k = 0; k < V; ++k) acc.e[k] += v[u].e[k];
        }
    }
    if (cur < A.vocab) {
        if (first && open_head) {         // the whole chunk: one entry, continued to the right if it goes on
            k0 = cur;
            f0 = 1;
            if (on) stv<float, V>(A.nsrc + (2 * c) * A.dim + j, acc);
            if (open_tail) k1 = cur;
        } else if (open_tail) {
            k1 = cur;
            f1 = 1;
            if (on) stv<float, V>(A.nsrc + (2 * c + 1) * A.dim + j, acc);
        } else if (on) {
#pragma unroll
            for (int k = 0; k < V; ++k) acc.e[k] *= A.scale;
            stv<T, V>(out + (long long)cur * A.dim, acc);
        }
    }
    if (lane == 0 && (A.own_entries || blockIdx.y == 0) && A.nentry) {
        A.nentry[2 * c] = make_uint2(k0, f0);
        A.nentry[2 * c + 1] = make_uint2(k1, f1);
    }
}

template <class T, class S, int V, bool LEAF> __global__ __launch_bounds__(256) void seg_sum_kernel(const SegArgs A) {
    const long long c = (long long)blockIdx.x * (256 >> A.w_log) + (threadIdx.x >> A.w_log);
    if (c * A.chunk < A.n) seg_chunk<T, S, V, LEAF>(A, c, threadIdx.x & (A.W - 1));
}

// All levels from one of at most kTailEntries entries on, in one block per block of columns: they are a few
// chunks each and a launch apiece would cost more than the sums.  Two sets of entries and rows take turns;
// every block of columns keeps its own copy of the entries (the same in all).
constexpr int kTailEntries = 1024;
struct SegTail {
    uint2 *entry[2];      // [column blocks][2 * chunks of the first level]
    float *src[2];
};
template <class T, int V> __global__ __launch_bounds__(256) void seg_tail_kernel(SegArgs A, const SegTail B) {
    const int lane = threadIdx.x & (A.W - 1), groups = 256 >> A.w_log;
    const long long most = 2 * ((A.n + A.chunk - 1) / A.chunk);
    for (int l = 0;; l ^= 1) {
        const long long chunks = (A.n + A.chunk - 1) / A.chunk;
        A.nentry = chunks > 1 ? B.entry[l] + blockIdx.y * most : nullptr;
        A.nsrc = B.src[l];
        for (long long c = threadIdx.x >> A.w_log; c < chunks; c += groups) seg_chunk<T, float, V, false>(A, c, lane);
        if (chunks <= 1) return;
        __syncthreads();          // the next level reads what this block stored
        A.entry = A.nentry;
        A.src = A.nsrc;
        A.n = 2 * chunks;
    }
}

__global__ __launch_bounds__(256) void emb_zero_kernel(char *p, long long bytes) { zero_fill(p, bytes, blockIdx.x, gridDim.x); }

constexpr int kMaxLevels = 10;
struct EmbGeom {
    long long n;
    int blocks, passes, bits, items, chunk0, chunk, levels;
    long long entries[kMaxLevels + 1];    // of each level; level 0 = n
};

static EmbGeom emb_geom(long long n, long long vocab) {
    EmbGeom G;
    memset(&G, 0, sizeof(G));
    G.n = n;
    int bits = 1;
    while (bits < 32 && (1ll << bits) <= vocab) ++bits;      // keys 0 .. vocab
    const bool small = n <= kSmallSort;
    G.passes = small ? (bits + 7) / 8 : (bits + kSortMaxBits - 1) / kSortMaxBits;
    G.bits = small ? 8 : (bits + G.passes - 1) / G.passes;
    // tiles of 4096 items, of 1024 where those would leave compute units idle
    G.items = n >= (1 << 20) ? 16 : 4;
    G.blocks = (int)((n + 256ll * G.items - 1) / (256ll * G.items));
    // long chunks leave fewer ends to sum again, short ones keep the chip busy when there are few rows
    G.chunk0 = n >= (1 << 20) || n <= 64 ? 64 : (n >= (1 << 17) ? 32 : 16);
    G.chunk = 32;
    G.entries[0] = n;
    G.levels = 1;
    for (long long c = (n + G.chunk0 - 1) / G.chunk0; c > 1; c = (2 * c + G.chunk - 1) / G.chunk) {
        G.entries[G.levels] = 2 * c;
        ++G.levels;
        if (2 * c <= kTailEntries) break;      // the tail kernel takes it from here
    }
    return G;
}

static int emb_check(int32_t dtype, int64_t n, int64_t vocab, int64_t dim) {
    GATMI_REQUIRE(dtype >= GATMI_F32 && dtype <= GATMI_F16, "embedding: unknown element type %d", dtype);
    GATMI_REQUIRE(n >= 0 && n < (1ll << 31) && vocab >= 0 && vocab < (1ll << 31) && dim >= 1 && dim <= 65536,
                  "embedding: %lld ids, %lld rows of %lld out of range", (long long)n, (long long)vocab, (long long)dim);
    return GATMI_OK;
}

static int emb_lanes(int v, int64_t dim) {
    const long long nv = (dim + v - 1) / v;
    return nv >= 64 ? 64 : next_pow2((int)nv);
}

}  // namespace gatmi

using namespace gatmi;

extern "C" int gatmi_embedding_fwd(int32_t dtype, int64_t n, int64_t vocab, int64_t dim, float scale,
                                   const int64_t *ids, const void *table, void *y, void *stream) {
    if (int e = emb_check(dtype, n, vocab, dim)) return e;
    if (n == 0) return GATMI_OK;
    GATMI_REQUIRE(ids && (table || vocab == 0) && y, "embedding_fwd: null argument");
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int v = vec_of(dtype, dim);
    EmbArgs A{ids, table, y, n, vocab, (int)dim, emb_lanes(v, dim), 0, scale};
    A.w_log = ilog2(A.W);
    const long long per = (256 >> A.w_log) * kEmbUnroll;
    ProfScope ps("embedding_fwd", st);
    // a launch counts its threads in 32 bits: 2^23 blocks of 256 at most
    for (long long i = 0; i < n; i += per << 23) {
        A.ids = ids + i;
        A.n = n - i < per << 23 ? n - i : per << 23;
        GATMI_WITH_TYPE(dtype, {
            A.y = static_cast<T *>(y) + i * dim;
            with_vec<T>(v, [&](auto V) {
                hipLaunchKernelGGL((emb_fwd_kernel<T, decltype(V)::value>), dim3((unsigned)((A.n + per - 1) / per)),
                                   dim3(256), 0, st, A);
            });
        });
    }
    GATMI_HIP(hipGetLastError());
    return GATMI_OK;
}

struct EmbWs {
    uint2 *pair[2], *lentry[2], *tentry[2];
    uint32_t *hist, *total;
    float *lsrc[2], *tsrc[2];
    size_t bytes;
};
static EmbWs emb_carve(const EmbGeom &G, long long dim, void *ws) {
    Carver cv(ws);
    EmbWs w;
    for (int i = 0; i < 2; ++i) w.pair[i] = cv.take<uint2>(G.n);
    w.hist = cv.take<uint32_t>((1ll << G.bits) * G.blocks);
    w.total = cv.take<uint32_t>(1ll << G.bits);
    for (int i = 0; i < 2; ++i) {        // levels 1, 3, .. and 2, 4, ..
        const long long m = G.levels > 1 + i ? G.entries[1 + i] : 0;
        w.lentry[i] = cv.take<uint2>(m);
        w.lsrc[i] = cv.take<float>(m * dim);
        // the tail's own: what its first level leaves is the most
        const long long t = G.levels > 1 ? 2 * ((G.entries[G.levels - 1] + G.chunk - 1) / G.chunk) : 0;
        w.tentry[i] = cv.take<uint2>(t * ((dim + 63) / 64));
        w.tsrc[i] = cv.take<float>(t * dim);
    }
    w.bytes = cv.off + 256;
    return w;
}

extern "C" size_t gatmi_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t dim) {
    if (emb_check(GATMI_F32, n, vocab, dim)) return 0;
    return emb_carve(emb_geom(n, vocab), dim, nullptr).bytes;
}

extern "C" int gatmi_embedding_bwd(int32_t dtype, int64_t n, int64_t vocab, int64_t dim, float scale,
                                   const int64_t *ids, const void *grad_y, void *grad_table, void *ws,
                                   size_t ws_bytes, void *stream) {
    if (int e = emb_check(dtype, n, vocab, dim)) return e;
    if (vocab == 0) return GATMI_OK;
    GATMI_REQUIRE(grad_table && (n == 0 || (ids && grad_y)), "embedding_bwd: null argument");
    const EmbGeom G = emb_geom(n, vocab);
    const EmbWs w = emb_carve(G, dim, ws);
    if (ws_bytes < w.bytes || !ws) {
        set_error("embedding workspace too small: %zu < %zu", ws_bytes, w.bytes);
        return GATMI_ERR_WS;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    // every row is cleared, then the rows that have ids are stored
    const long long clear = vocab * dim * (dtype == GATMI_F32 ? 4 : 2);
    const unsigned clear_blocks = (unsigned)(clear / 16384 < 1 ? 1 : (clear / 16384 > 8192 ? 8192 : clear / 16384));
    if (n == 0 || n > kSmallSort) {
        ProfScope ps("embedding_zero", st);
        hipLaunchKernelGGL(emb_zero_kernel, dim3(clear_blocks), dim3(256), 0, st, static_cast<char *>(grad_table), clear);
        GATMI_HIP(hipGetLastError());
    }
    if (n == 0) return GATMI_OK;
    {
        ProfScope ps("embedding_sort", st);
        SortArgs S;
        memset(&S, 0, sizeof(S));
        S.n = n;
        S.vocab = vocab;
        S.blocks = G.blocks;
        S.hist = w.hist;
        S.total = w.total;
        S.bits = G.bits;
        S.passes = G.passes;
        if (n <= kSmallSort) {
            S.ids = ids;
            S.out = w.pair[(G.passes - 1) & 1];
            hipLaunchKernelGGL(sort_small_kernel, dim3(1 + clear_blocks), dim3(256), 0, st, S,
                               static_cast<char *>(grad_table), clear);
        }
        for (int p = 0; n > kSmallSort && p < G.passes; ++p) {
            const size_t bins = (size_t)1 << G.bits;
            S.ids = p == 0 ? ids : nullptr;
            S.in = w.pair[(p + 1) & 1];
            S.out = w.pair[p & 1];
            S.shift = G.bits * p;
            auto count = G.items == 16 ? sort_count_kernel<16> : sort_count_kernel<4>;
            auto scatter = G.items == 16 ? sort_scatter_kernel<16> : sort_scatter_kernel<4>;
            hipLaunchKernelGGL(count, dim3(G.blocks), dim3(256), bins * 4, st, S);
            hipLaunchKernelGGL(sort_scan_kernel, dim3((unsigned)bins), dim3(256), 0, st, S);
            hipLaunchKernelGGL(scatter, dim3(G.blocks), dim3(256), bins * 20 + 2048ll * G.items, st, S);
        }
        GATMI_HIP(hipGetLastError());
    }
    ProfScope ps("embedding_sum", st);
    const int last = (G.passes - 1) & 1;
    SegArgs A;
    memset(&A, 0, sizeof(A));
    A.vocab = (uint32_t)vocab;
    A.dim = (int)dim;
    A.scale = scale;
    A.out = grad_table;
    for (int l = 0; l < G.levels; ++l) {
        A.n = G.entries[l];
        A.chunk = l == 0 ? G.chunk0 : G.chunk;
        A.entry = l == 0 ? w.pair[last] : w.lentry[(l - 1) & 1];
        A.src = l == 0 ? grad_y : w.lsrc[(l - 1) & 1];
        const bool more = l + 1 < G.levels, tail = l > 0 && !more;
        A.nentry = more ? w.lentry[l & 1] : nullptr;
        A.nsrc = w.lsrc[l & 1];
        // f32 partial rows take vectors of their own width
        const int v = l == 0 ? vec_of(dtype, dim) : vec_of(GATMI_F32, dim);
        A.W = emb_lanes(v, dim);
        A.w_log = ilog2(A.W);
        const long long chunks = (A.n + A.chunk - 1) / A.chunk, per = 256 >> A.w_log;
        const dim3 grid((unsigned)((chunks + per - 1) / per), (unsigned)((dim + (long long)A.W * v - 1) / ((long long)A.W * v)));
        const SegTail B{{w.tentry[0], w.tentry[1]}, {w.tsrc[0], w.tsrc[1]}};
        A.own_entries = tail;
        GATMI_WITH_TYPE(dtype, {
            if (tail)
                with_vec<float>(v, [&](auto V) {
                    hipLaunchKernelGGL((seg_tail_kernel<T, decltype(V)::value>), dim3(1, grid.y), dim3(256), 0, st, A, B);
                });
            else if (l == 0)
                with_vec<T>(v, [&](auto V) {
                    hipLaunchKernelGGL((seg_sum_kernel<T, T, decltype(V)::value, true>), grid, dim3(256), 0, st, A);
                });
            else
                with_vec<float>(v, [&](auto V) {
                    hipLaunchKernelGGL((seg_sum_kernel<T, float, decltype(V)::value, false>), grid, dim3(256), 0, st, A);
                });
        });
        GATMI_HIP(hipGetLastError());
    }
    return GATMI_OK;
}
