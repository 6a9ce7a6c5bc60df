// The complex embedding lookup with scaling, and its gradient by sorted tokens.
//
// Forward (ComplexEmbed.forward, v11/complex_ops.py:223-235):
//   out[n][j] = scale (re[id_n][j], im[id_n][j]),  interleaved [n][dim][2];
// a row of a given value (`outside`) where id_n is no row of the table.
// Backward:
//   d re[v][j] = scale sum_{n: id_n = v} dz[n][j][0],  d im from dz[n][j][1],
// dense [V][dim] tables: tokens that do not occur get zeros.
//
// The sum of a token runs over its positions in ascending order, in fp32, so the
// gradient is the same bits on every call: a stable radix sort of the ids gives
// the positions of each token in order, and the sorted list is cut into chunks of
// CH entries.  A run of equal tokens inside one chunk is summed and written by
// that chunk; a run that crosses chunks leaves a partial sum in each, which a
// second pass adds in chunk order.
#include <algorithm>

#include "common.h"

namespace qpam {
namespace embed {
namespace {

constexpr int THREADS = 256;
constexpr int RADIX_BITS = 8, RADIX = 1 << RADIX_BITS;

// one rounding to the table's type; infinities and NaN stay what they are
template <typename T> __device__ __forceinline__ T to_elem(float x);
template <> __device__ __forceinline__ float to_elem<float>(float x) { return x; }
template <> __device__ __forceinline__ unsigned short to_elem<unsigned short>(float x) {
    return __builtin_bit_cast(unsigned short, (__bf16)x);
}

__device__ __forceinline__ int64_t load_id(const void *ids, int is64, int64_t i) {
    return is64 ? static_cast<const int64_t *>(ids)[i] : static_cast<const int32_t *>(ids)[i];
}

// ---------------------------------------------------------------- lookup ---
// W complex values of one table row per lane and step: 16 bytes of each table in, two
// 16-byte stores out.  Lanes to a row: the least power of two that covers it, at most a
// wave, so that short rows share waves.  PAIRS: one interleaved table [V][dim][2] (im = re + 1,
// columns two apart), whose rows are the output's form already.  W = 1: any column strides.  Bound by the launch (192 rows of 768 fp32: 3.3
// us) or by gathering and storing: 16384 rows of 512 bf16 12.4 us, 33 MB written and 12 MB of
// distinct rows read (3.7 TB/s; a frequent token's row comes from the caches).
template <typename T, int W, bool PAIRS>
__global__ void __launch_bounds__(THREADS) lookup_kernel(qpam_embed_args a, int lanes_log2) {
    typedef T VecT __attribute__((ext_vector_type(W)));
    const int lanes = 1 << lanes_log2;  // lanes that share a row
    const int64_t gid = (int64_t)blockIdx.x * THREADS + threadIdx.x;
    const int64_t row = gid >> lanes_log2;
    if (row >= a.n) return;
    const int64_t id = load_id(a.ids, a.ids_i64, row);
    const bool ok = id >= 0 && id < a.V;
    const T *re = static_cast<const T *>(a.re) + (ok ? id : 0) * a.ld_re;
    const T *im = static_cast<const T *>(a.im) + (ok ? id : 0) * a.ld_im;
    T *out = static_cast<T *>(a.out) + row * 2 * a.dim;
    for (int j = W * (int)(gid & (lanes - 1)); j < a.dim; j += W * lanes) {
        alignas(16) T x[2 * W], o[2 * W];  // PAIRS: as they stand; otherwise the reals, then the imaginaries
        if constexpr (PAIRS) {
            *reinterpret_cast<VecT *>(x) = *reinterpret_cast<const VecT *>(re + 2 * j);
            *reinterpret_cast<VecT *>(x + W) = *reinterpret_cast<const VecT *>(re + 2 * j + W);
        } else if constexpr (W > 1) {
            *reinterpret_cast<VecT *>(x) = *reinterpret_cast<const VecT *>(re + j);
            *reinterpret_cast<VecT *>(x + W) = *reinterpret_cast<const VecT *>(im + j);
        } else {
            x[0] = re[j * a.cs_re];
            x[1] = im[j * a.cs_im];
        }
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) o[i] = to_elem<T>(ok ? Elem<T>::load(x + (PAIRS ? i : i / 2 + i % 2 * W)) * a.scale : a.outside);
        if constexpr (W > 1) {
            uintx4 *dst = reinterpret_cast<uintx4 *>(out + 2 * j);
            dst[0] = reinterpret_cast<const uintx4 *>(o)[0];
            dst[1] = reinterpret_cast<const uintx4 *>(o)[1];
        } else {
            out[2 * j] = o[0];
            out[2 * j + 1] = o[1];
        }
    }
}

// ------------------------------------------------------------------ sort ---
// Sorted list: key = token, or V for a position without a gradient (padding token
// or an id outside the table), which sorts behind every token.
struct SortParams {
    qpam_embed_args a;
    int n;
    uint32_t *key, *pos;    // the list this launch reads (NULL: the ids themselves)
    uint32_t *key2, *pos2;  // ... and writes
    uint32_t *hist;         // [RADIX][tiles]
    int tiles, shift;
    int64_t fill16;         // 16-byte units of each gradient table, or 0
    int sort_blocks;        // blocks that sort; the others zero the tables
};

__device__ __forceinline__ uint32_t key_of(const qpam_embed_args &a, int64_t i) {
    const int64_t id = load_id(a.ids, a.ids_i64, i);
    return (id >= 0 && id < a.V && id != a.padding_idx) ? (uint32_t)id : (uint32_t)a.V;
}

// Lanes of the wave (of `active`) with this lane's digit.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, uint64_t active) {
    uint64_t m = active;
#pragma unroll
    for (int b = 0; b < RADIX_BITS; ++b) {
        const bool bit = (digit >> b) & 1;
        const uint64_t bal = __ballot(bit);
        m &= bit ? bal : ~bal;
    }
    return m;
}

// Blocks beyond the sorting ones write zeros over both tables (16-byte units, then
// the tail elements by the first of them).
__device__ __forceinline__ void zero_tables(const SortParams &p) {
    const int64_t nb = gridDim.x - p.sort_blocks, b = blockIdx.x - p.sort_blocks;
    const int64_t bytes = (int64_t)p.a.V * p.a.dim * (p.a.dtype == QPAM_F32 ? 4 : 2);
    const uintx4 z = {0u, 0u, 0u, 0u};
    for (int t = 0; t < 2; ++t) {
        char *base = static_cast<char *>(t ? p.a.d_im : p.a.d_re);
        uintx4 *d = reinterpret_cast<uintx4 *>(base);
        for (int64_t i = b * blockDim.x + threadIdx.x; i < p.fill16; i += nb * blockDim.x) d[i] = z;
        if (b == 0)
            for (int64_t i = 16 * p.fill16 + threadIdx.x * 2; i < bytes; i += blockDim.x * 2)
                *reinterpret_cast<unsigned short *>(base + i) = 0;
    }
}

// Up to SMALL ids sorted by one block: the list lives in LDS between the passes,
// each wave ranks a contiguous part of it (stable: rounds of 64 in order, lanes of
// a round in order), and the counts of [wave][digit] give every wave its places.
// One launch instead of the six of the longer lists' two passes, and the other blocks
// zero the tables beside it: 37 us for 16384 ids and 103 MB (the sort's own time; the
// fill alone takes 15), 27 us for 3001 ids and 197 MB (the fill's).
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr int ROUNDS = 16, SMALL = SORT_THREADS * ROUNDS;
constexpr size_t SORT_SMEM = SMALL * 6 + SORT_WAVES * RADIX * 4;

__global__ void __launch_bounds__(SORT_THREADS) sort_small_kernel(SortParams p, int passes) {
    if ((int)blockIdx.x >= p.sort_blocks) {
        zero_tables(p);
        return;
    }
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ uint32_t wsum[4];
    uint32_t *sKey = reinterpret_cast<uint32_t *>(smem);
    unsigned short *sPos = reinterpret_cast<unsigned short *>(smem + SMALL * 4);
    uint32_t *sHist = reinterpret_cast<uint32_t *>(smem + SMALL * 6);  // [wave][digit]
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int rounds = (p.n + SORT_THREADS - 1) / SORT_THREADS;
    const int first = w * rounds * 64;
    for (int i = tid; i < p.n; i += SORT_THREADS) {
        sKey[i] = key_of(p.a, i);
        sPos[i] = (unsigned short)i;
    }
    uint32_t *hw = sHist + w * RADIX;
    for (int pass = 0; pass < passes; ++pass) {
        for (int i = lane; i < RADIX; i += 64) hw[i] = 0;
        __syncthreads();
        uint32_t key[ROUNDS], rank[ROUNDS];
        unsigned short pos[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            if (r >= rounds) continue;
            const int i = first + 64 * r + lane;
            const bool on = i < p.n;
            key[r] = on ? sKey[i] : 0u;
            pos[r] = on ? sPos[i] : (unsigned short)0;
            const uint32_t digit = (key[r] >> (RADIX_BITS * pass)) & (RADIX - 1);
            const uint64_t m = same_digit(digit, __ballot(on));
            const uint32_t before = __popcll(m & ((1ull << lane) - 1));
            const uint32_t base = hw[digit];
            wave_lds_order();
            if (on && before == 0) hw[digit] = base + __popcll(m);
            wave_lds_order();
            rank[r] = base + before;
        }
        __syncthreads();
        uint32_t total = 0, at = 0;
        if (tid < RADIX) {
            for (int v = 0; v < SORT_WAVES; ++v) {
                const uint32_t c = sHist[v * RADIX + tid];
                sHist[v * RADIX + tid] = total;
                total += c;
            }
            at = total;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const uint32_t o = __shfl_up(at, off);
                if (lane >= off) at += o;
            }
            if (lane == 63) wsum[w] = at;
        }
        __syncthreads();
        if (tid < RADIX) {
            at -= total;  // exclusive
            for (int v = 0; v < w; ++v) at += wsum[v];
            for (int v = 0; v < SORT_WAVES; ++v) sHist[v * RADIX + tid] += at;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            if (r >= rounds || first + 64 * r + lane >= p.n) continue;
            const uint32_t digit = (key[r] >> (RADIX_BITS * pass)) & (RADIX - 1);
            const uint32_t to = hw[digit] + rank[r];
            sKey[to] = key[r];
            sPos[to] = pos[r];
        }
        __syncthreads();
    }
    for (int i = tid; i < p.n; i += SORT_THREADS) {
        p.key2[i] = sKey[i];
        p.pos2[i] = sPos[i];
    }
}

// Longer lists, one pass of the sort in three launches: counts per tile and digit,
// a scan of each digit's counts over the tiles, and the placement.
constexpr int TILE = 4096, TROUNDS = TILE / THREADS, TWAVES = THREADS / 64;

__device__ __forceinline__ uint32_t list_key(const SortParams &p, int i) { return p.key ? p.key[i] : key_of(p.a, i); }

__global__ void __launch_bounds__(THREADS) hist_kernel(SortParams p) {
    if ((int)blockIdx.x >= p.sort_blocks) {
        zero_tables(p);
        return;
    }
    __shared__ uint32_t h[RADIX];
    h[threadIdx.x] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * TILE;
    for (int r = 0; r < TROUNDS; ++r) {
        const int64_t i = base + r * THREADS + threadIdx.x;
        if (i < p.n) atomicAdd(&h[(list_key(p, (int)i) >> p.shift) & (RADIX - 1)], 1u);
    }
    __syncthreads();
    p.hist[(int64_t)threadIdx.x * p.tiles + blockIdx.x] = h[threadIdx.x];
}

// one block per digit: hist[digit][tile] -> exclusive prefix over the tiles; the
// digit's total goes behind the table, hist[RADIX tiles + digit]
__global__ void __launch_bounds__(THREADS) scan_kernel(SortParams p) {
    __shared__ uint32_t wsum[TWAVES];
    uint32_t *h = p.hist + (int64_t)blockIdx.x * p.tiles;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int t0 = 0; t0 < p.tiles; t0 += THREADS) {
        const int t = t0 + threadIdx.x;
        const uint32_t c = t < p.tiles ? h[t] : 0u;
        uint32_t at = c;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(at, off);
            if (lane >= off) at += o;
        }
        if (lane == 63) wsum[w] = at;
        __syncthreads();
        uint32_t before = carry, all = 0;
        for (int v = 0; v < TWAVES; ++v) {
            if (v < w) before += wsum[v];
            all += wsum[v];
        }
        if (t < p.tiles) h[t] = before + at - c;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) p.hist[(int64_t)RADIX * p.tiles + blockIdx.x] = carry;
}

__global__ void __launch_bounds__(THREADS) place_kernel(SortParams p) {
    __shared__ uint32_t sHist[TWAVES][RADIX], wsum[TWAVES];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
    const int64_t first = (int64_t)blockIdx.x * TILE + w * (TILE / TWAVES);
    for (int i = tid; i < TWAVES * RADIX; i += THREADS) (&sHist[0][0])[i] = 0;
    __syncthreads();
    uint32_t key[TROUNDS], rank[TROUNDS];
#pragma unroll
    for (int r = 0; r < TROUNDS; ++r) {
        const int64_t i = first + 64 * r + lane;
        const bool on = i < p.n;
        key[r] = on ? list_key(p, (int)i) : 0u;
        const uint32_t digit = (key[r] >> p.shift) & (RADIX - 1);
        const uint64_t m = same_digit(digit, __ballot(on));
        const uint32_t before = __popcll(m & ((1ull << lane) - 1));
        const uint32_t base = sHist[w][digit];
        wave_lds_order();
        if (on && before == 0) sHist[w][digit] = base + __popcll(m);
        wave_lds_order();
        rank[r] = base + before;
    }
    __syncthreads();
    {   // thread = digit: where the digit's entries of this tile begin, then of each wave
        const uint32_t total = p.hist[(int64_t)RADIX * p.tiles + tid];
        uint32_t at = total;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t o = __shfl_up(at, off);
            if (lane >= off) at += o;
        }
        if (lane == 63) wsum[w] = at;
        __syncthreads();
        at -= total;
        for (int v = 0; v < w; ++v) at += wsum[v];
        at += p.hist[(int64_t)tid * p.tiles + blockIdx.x];
        for (int v = 0; v < TWAVES; ++v) {
            const uint32_t c = sHist[v][tid];
            sHist[v][tid] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < TROUNDS; ++r) {
        const int64_t i = first + 64 * r + lane;
        if (i >= p.n) continue;
        const uint32_t to = sHist[w][(key[r] >> p.shift) & (RADIX - 1)] + rank[r];
        p.key2[to] = key[r];
        p.pos2[to] = p.pos ? p.pos[i] : (uint32_t)i;
    }
}

// -------------------------------------------------------------- gradient ---
constexpr int CH = 16;  // sorted entries of a chunk

struct GradParams {
    qpam_embed_args a;
    int n, chunks, segs;   // segs: column segments of 64 lanes
    const uint32_t *key, *pos;
    float *part;           // [chunks][2][2 dim]: the run from the chunk before, the run into the next
};

template <typename T, int W>
__device__ __forceinline__ void write_row(const GradParams &p, uint32_t key, int j, const float *acc) {
    typedef T VecT __attribute__((ext_vector_type(W)));
    T r[W], m[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        r[i] = to_elem<T>(acc[2 * i] * p.a.scale);
        m[i] = to_elem<T>(acc[2 * i + 1] * p.a.scale);
    }
    const int64_t o = (int64_t)key * p.a.dim + j;
    *reinterpret_cast<VecT *>(static_cast<T *>(p.a.d_re) + o) = *reinterpret_cast<const VecT *>(r);
    *reinterpret_cast<VecT *>(static_cast<T *>(p.a.d_im) + o) = *reinterpret_cast<const VecT *>(m);
}

// One wave: a chunk's entries over 64 W complex columns, 8 bytes of a table's row a lane.
// Bound by the latency of its gathered rows, so all CH are in flight at once; a longer
// chunk has fewer waves, a shorter one more partial sums.  16384 rows of 512 bf16 (33 MB
// read): 12.0 us, and 4.3 us for the runs that cross chunks.
template <typename T, int W>
__global__ void __launch_bounds__(THREADS) grad_chunk_kernel(GradParams p) {
    typedef T VecT __attribute__((ext_vector_type(2 * W)));
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * (THREADS / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (item >= (int64_t)p.chunks * p.segs) return;
    const int c = (int)(item / p.segs), seg = (int)(item - (int64_t)c * p.segs);
    const int j = W * (64 * seg + lane);
    const bool on = j < p.a.dim;
    const int e0 = c * CH, cnt = min(CH, p.n - e0);
    // lane l holds entry e0 - 1 + l of the list
    const int mine = min(max(e0 - 1 + lane, 0), p.n - 1);
    const uint32_t keys = lane <= CH + 1 ? p.key[mine] : 0u, poss = lane <= CH + 1 ? p.pos[mine] : 0u;
    const T *dz = static_cast<const T *>(p.a.dz) + 2 * (on ? j : 0);
    // every row of the chunk in flight at once (entries past the list's end re-read its
    // last one); the empty asm keeps the compiler from moving a load down to its use
    VecT x[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t pos = __builtin_amdgcn_readlane(poss, i + 1);
        x[i] = *reinterpret_cast<const VecT *>(dz + (int64_t)pos * 2 * p.a.dim);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) asm volatile("" : "+v"(x[i]));
    const uint32_t V = (uint32_t)p.a.V;
    float acc[2 * W];
#pragma unroll
    for (int k = 0; k < 2 * W; ++k) acc[k] = 0.f;
    uint32_t cur = __builtin_amdgcn_readlane(keys, 1);
    bool starts = c == 0 || (uint32_t)__builtin_amdgcn_readlane(keys, 0) != cur;
    auto flush = [&](bool ends) {
        if (cur >= V || !on) return;
        if (starts && ends) {
            write_row<T, W>(p, cur, j, acc);
        } else {
            float *dst = p.part + ((int64_t)c * 2 + (starts ? 1 : 0)) * 2 * p.a.dim + 2 * j;
#pragma unroll
            for (int k = 0; k < 2 * W; ++k) dst[k] = acc[k];
        }
    };
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (i >= cnt) continue;
        const uint32_t k = __builtin_amdgcn_readlane(keys, i + 1);
        if (k != cur) {
            flush(true);
            cur = k;
            starts = true;
#pragma unroll
            for (int t = 0; t < 2 * W; ++t) acc[t] = 0.f;
        }
        T v[2 * W];
        *reinterpret_cast<VecT *>(v) = x[i];
#pragma unroll
        for (int t = 0; t < 2 * W; ++t) acc[t] += Elem<T>::load(v + t);
    }
    flush(e0 + cnt >= p.n || (uint32_t)__builtin_amdgcn_readlane(keys, CH + 1) != cur);
}

// A run that begins in chunk c and goes on: its partial sums in chunk order, each
// of the block's waves a contiguous part of them.
template <typename T, int W>
__global__ void __launch_bounds__(THREADS) grad_runs_kernel(GradParams p) {
    constexpr int WAVES = THREADS / 64;
    __shared__ float sPart[WAVES][64 * 2 * W];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = blockIdx.x / p.segs, seg = blockIdx.x - c * p.segs;
    if (c + 1 >= p.chunks) return;
    const int last = (c + 1) * CH - 1;
    const uint32_t key = p.key[last];
    if (key >= (uint32_t)p.a.V || p.key[last + 1] != key) return;
    if (p.key[c * CH] == key && c > 0 && p.key[c * CH - 1] == key) return;  // begins before this chunk
    // chunks after c whose first entry is still the run's
    int len = 0;
    for (;;) {
        const int64_t cc = (int64_t)c + 1 + len + lane;
        const uint64_t m = __ballot(cc < p.chunks && p.key[min(cc * CH, (int64_t)p.n - 1)] == key);
        const int k = m == ~0ull ? 64 : __ffsll((unsigned long long)~m) - 1;
        len += k;
        if (k < 64) break;
    }
    const int j = W * (64 * seg + lane);
    const bool on = j < p.a.dim;
    // partial i: 0 is chunk c's own, i > 0 chunk c + i's
    const int total = len + 1, per = (total + WAVES - 1) / WAVES;
    const int i0 = w * per, i1 = min(total, i0 + per);
    float acc[2 * W];
#pragma unroll
    for (int k = 0; k < 2 * W; ++k) acc[k] = 0.f;
    if (on) {
#pragma unroll 4
        for (int i = i0; i < i1; ++i) {
            const float *src = p.part + ((int64_t)(c + i) * 2 + (i == 0 ? 1 : 0)) * 2 * p.a.dim + 2 * j;
#pragma unroll
            for (int k = 0; k < 2 * W; ++k) acc[k] += src[k];
        }
    }
#pragma unroll
    for (int k = 0; k < 2 * W; ++k) sPart[w][k * 64 + lane] = acc[k];
    __syncthreads();
    if (w == 0 && on) {
#pragma unroll
        for (int k = 0; k < 2 * W; ++k)
            for (int v = 1; v < WAVES; ++v) acc[k] += sPart[v][k * 64 + lane];
        write_row<T, W>(p, key, j, acc);
    }
}

// ------------------------------------------------------------------ host ---
constexpr int64_t MAX_N = (int64_t)1 << 30;
constexpr int64_t MAX_THREADS = (int64_t)1 << 31;  // of a launch, which holds less than 2^32

struct Layout {
    size_t list[2], hist, part, bytes;
    int tiles, chunks;
};

Layout layout(int64_t n, int dim) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    Layout l;
    l.tiles = (int)((n + TILE - 1) / TILE);
    l.chunks = (int)((n + CH - 1) / CH);
    size_t at = 0;
    l.list[0] = at;
    at += up((size_t)n * 8);
    l.list[1] = at;
    if (n > SMALL) at += up((size_t)n * 8);
    l.hist = at;
    if (n > SMALL) at += up(((size_t)RADIX * l.tiles + RADIX) * 4);
    l.part = at;
    at += up((size_t)l.chunks * 2 * 2 * dim * 4);
    l.bytes = at;
    return l;
}

int check(const qpam_embed_args &a, const char *who) {
    QPAM_REQUIRE(a.dtype == QPAM_F32 || a.dtype == QPAM_BF16, "%s: dtype %d", who, a.dtype);
    QPAM_REQUIRE(a.n >= 0 && a.n <= MAX_N, "%s: %lld ids (at most 2^30)", who, (long long)a.n);
    QPAM_REQUIRE(a.V >= 1 && a.V < (1 << 30) && a.dim >= 1 && a.dim <= (1 << 20), "%s: table %d x %d", who, a.V, a.dim);
    QPAM_REQUIRE(a.n == 0 || a.ids, "%s: null ids", who);
    return QPAM_OK;
}

template <typename T>
int run_lookup(const qpam_embed_args &a, hipStream_t stream) {
    constexpr int W = 16 / sizeof(T);
    const bool rows = a.dim % W == 0 && a.ld_re % W == 0 && ((uintptr_t)a.re % 16) == 0 && ((uintptr_t)a.out % 16) == 0;
    const bool planes = rows && a.cs_re == 1 && a.cs_im == 1 && a.ld_im % W == 0 && ((uintptr_t)a.im % 16) == 0;
    const bool pairs = rows && a.cs_re == 2 && a.cs_im == 2 && a.ld_im == a.ld_re && a.im == static_cast<const T *>(a.re) + 1;
    const bool wide = planes || pairs;
    const int steps = wide ? a.dim / W : a.dim;
    int lg = 0;
    while (lg < 6 && (1 << lg) < steps) ++lg;
    const int64_t per = MAX_THREADS >> lg;  // rows of a launch
    for (int64_t n0 = 0; n0 < a.n; n0 += per) {
        qpam_embed_args s = a;
        s.n = std::min(per, a.n - n0);
        s.ids = static_cast<const char *>(a.ids) + n0 * (a.ids_i64 ? 8 : 4);
        s.out = static_cast<T *>(a.out) + n0 * 2 * a.dim;
        const unsigned blocks = (unsigned)(((s.n << lg) + THREADS - 1) / THREADS);
        if (pairs)
            hipLaunchKernelGGL((lookup_kernel<T, W, true>), dim3(blocks), dim3(THREADS), 0, stream, s, lg);
        else if (planes)
            hipLaunchKernelGGL((lookup_kernel<T, W, false>), dim3(blocks), dim3(THREADS), 0, stream, s, lg);
        else
            hipLaunchKernelGGL((lookup_kernel<T, 1, false>), dim3(blocks), dim3(THREADS), 0, stream, s, lg);
        const int st = launch_status("embed lookup_kernel");
        if (st) return st;
    }
    return QPAM_OK;
}

template <typename T, int W>
int launch_grad(const GradParams &g, hipStream_t stream) {
    const int64_t items = (int64_t)g.chunks * g.segs;
    hipLaunchKernelGGL((grad_chunk_kernel<T, W>), dim3((unsigned)((items + 3) / 4)), dim3(THREADS), 0, stream, g);
    int st = launch_status("embed grad_chunk_kernel");
    if (st || g.chunks < 2) return st;
    hipLaunchKernelGGL((grad_runs_kernel<T, W>), dim3((unsigned)items), dim3(THREADS), 0, stream, g);
    return launch_status("embed grad_runs_kernel");
}

template <typename T>
int run_grad(const qpam_embed_args &a, hipStream_t stream) {
    constexpr int W = 8 / sizeof(T);
    const bool wide = a.dim % W == 0;
    const Layout l = layout(a.n, a.dim);
    GradParams g;
    g.segs = (a.dim + 64 * (wide ? W : 1) - 1) / (64 * (wide ? W : 1));
    QPAM_REQUIRE((int64_t)l.chunks * g.segs * THREADS <= MAX_THREADS, "qpam_embed_bwd: too many ids for this dim");
    char *ws = static_cast<char *>(a.workspace);
    SortParams s;
    s.a = a;
    s.n = (int)a.n;
    s.key = s.pos = nullptr;
    s.hist = reinterpret_cast<uint32_t *>(ws + l.hist);
    s.tiles = l.tiles;
    s.shift = 0;
    const int64_t bytes = (int64_t)a.V * a.dim * sizeof(T);
    s.fill16 = bytes / 16;
    const int fill_blocks = (int)std::min<int64_t>(2048, (s.fill16 + 1023) / 1024 + 1);
    int bits = 0;
    while ((1u << bits) <= (unsigned)a.V) ++bits;
    const int passes = (bits + RADIX_BITS - 1) / RADIX_BITS;
    uint32_t *list[2] = {reinterpret_cast<uint32_t *>(ws + l.list[0]), reinterpret_cast<uint32_t *>(ws + l.list[1])};
    int st;
    int at = 0;  // the list that holds the result
    if (a.n <= SMALL) {
        s.sort_blocks = a.n > 0 ? 1 : 0;
        s.key2 = list[0];
        s.pos2 = list[0] + a.n;
        QPAM_CHECK_HIP(hipFuncSetAttribute((const void *)sort_small_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)SORT_SMEM));
        hipLaunchKernelGGL(sort_small_kernel, dim3(s.sort_blocks + fill_blocks), dim3(SORT_THREADS), SORT_SMEM, stream, s,
                           passes);
        st = launch_status("embed sort_small_kernel");
        if (st || a.n == 0) return st;
    } else {
        for (int pass = 0; pass < passes; ++pass) {
            at = pass & 1;
            s.key2 = list[at];
            s.pos2 = list[at] + a.n;
            s.shift = RADIX_BITS * pass;
            s.sort_blocks = l.tiles;
            hipLaunchKernelGGL(hist_kernel, dim3(l.tiles + (pass == 0 ? fill_blocks : 0)), dim3(THREADS), 0, stream, s);
            if ((st = launch_status("embed hist_kernel"))) return st;
            hipLaunchKernelGGL(scan_kernel, dim3(RADIX), dim3(THREADS), 0, stream, s);
            if ((st = launch_status("embed scan_kernel"))) return st;
            hipLaunchKernelGGL(place_kernel, dim3(l.tiles), dim3(THREADS), 0, stream, s);
            if ((st = launch_status("embed place_kernel"))) return st;
            s.key = s.key2;
            s.pos = s.pos2;
        }
    }
    g.a = a;
    g.n = (int)a.n;
    g.chunks = l.chunks;
    g.key = list[at];
    g.pos = list[at] + a.n;
    g.part = reinterpret_cast<float *>(ws + l.part);
    return wide ? launch_grad<T, W>(g, stream) : launch_grad<T, 1>(g, stream);
}

}  // namespace
}  // namespace embed
}  // namespace qpam

extern "C" int qpam_embed_fwd(const qpam_embed_args *a, void *stream) {
    using namespace qpam;
    using namespace qpam::embed;
    QPAM_REQUIRE(a != nullptr, "qpam_embed_fwd: null args");
    int st = check(*a, "qpam_embed_fwd");
    if (st || a->n == 0) return st;
    QPAM_REQUIRE(a->re && a->im && a->out, "qpam_embed_fwd: null table or output");
    auto fits = [&](int64_t ld, int64_t cs) { return cs >= 1 && cs <= ((int64_t)1 << 40) && ld > (a->dim - 1) * cs; };
    QPAM_REQUIRE(fits(a->ld_re, a->cs_re) && fits(a->ld_im, a->cs_im),
                 "qpam_embed_fwd: table column strides below 1, or row strides below a row");
    return a->dtype == QPAM_BF16 ? run_lookup<unsigned short>(*a, (hipStream_t)stream)
                                 : run_lookup<float>(*a, (hipStream_t)stream);
}

extern "C" size_t qpam_embed_bwd_workspace_size(const qpam_embed_args *a) {
    if (!a || a->n < 0 || a->n > qpam::embed::MAX_N || a->dim < 1) return 0;
    return qpam::embed::layout(a->n, a->dim).bytes;
}

extern "C" int qpam_embed_bwd(const qpam_embed_args *a, void *stream) {
    using namespace qpam;
    using namespace qpam::embed;
    QPAM_REQUIRE(a != nullptr, "qpam_embed_bwd: null args");
    int st = check(*a, "qpam_embed_bwd");
    if (st) return st;
    QPAM_REQUIRE(a->d_re && a->d_im && (a->n == 0 || a->dz), "qpam_embed_bwd: null dz, d_re or d_im");
    QPAM_REQUIRE(((uintptr_t)a->d_re % 16) == 0 && ((uintptr_t)a->d_im % 16) == 0 && ((uintptr_t)a->dz % 16) == 0,
                 "qpam_embed_bwd: dz and the gradient tables must be 16-byte aligned");
    const size_t need = qpam_embed_bwd_workspace_size(a);
    QPAM_REQUIRE(need == 0 || (a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace % 16) == 0),
                 "qpam_embed_bwd: workspace needs %zu bytes (got %zu)", need, a->workspace_bytes);
    return a->dtype == QPAM_BF16 ? run_grad<unsigned short>(*a, (hipStream_t)stream)
                                 : run_grad<float>(*a, (hipStream_t)stream);
}
