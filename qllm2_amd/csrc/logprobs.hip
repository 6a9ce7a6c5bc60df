// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits, and their gradient.
//
// With x the logits, T the temperature, m the row's maximum, u_v = (x_v - m) / T:
//   s = sum e^u,  t = sum e^u u,
//   logprob(v) = u_v - ln s,   entropy = ln s - t / s,
//   d x_v = ( g_lp ([v = token] - p_v) - g_ent p_v (ln p_v + entropy)
//             + sum_i g_top_i ([v = top_i] - p_v) ) / T.
// A row that a mask of -inf leaves empty (s = 0) has log probabilities -inf,
// entropy 0 and no gradient; a masked entry has p = 0 and adds nothing.
//
// Forward: one block per row and one pass over it.  Each thread keeps its own
// running maximum, s and t (rescaled when a batch of its entries raises the
// maximum) and the batch that holds its maximum; the block joins them.  u is taken
// in units of log2 so that e^u is one v_exp_f32, and the sums are fp32.
//
// Top alternatives without a sort or a second pass: the row's entries fall into 64
// groups (one per lane), the k-th largest of the groups' maxima bounds the k-th
// largest entry from below, and only the batches of 32 entries whose own maximum reaches
// that bound, about k, are read again (by the whole block) and the entries at or above it
// listed.  The list, about k long, is ranked by counting.  Entries order by value, equal
// values by the lower index, through one 64-bit key.
#include <algorithm>

#include "common.h"

namespace qpam {
namespace logprobs {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LOWEST = -3.402823466e38f;
// u of an entry that is -inf or far below the maximum: e^u is 0 and e^u u is -0, not NaN
constexpr float FLOOR = -1e4f;
constexpr int MAX_K = 64;
constexpr int CAP = 1024;  // listed candidates

typedef qpam_logprobs_args Args;

template <typename T> struct Vec {
    static constexpr int E = 16 / sizeof(T);
    __device__ __forceinline__ static void unpack(uintx4 r, float *x);
};
template <> __device__ __forceinline__ void Vec<float>::unpack(uintx4 r, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
}
template <> __device__ __forceinline__ void Vec<unsigned short>::unpack(uintx4 r, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(r[i] << 16);
        x[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
    }
}

// Order of values as unsigned integers: NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t order(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unorder(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint64_t make_key(float x, int idx) {
    return ((uint64_t)order(x) << 32) | (uint32_t)~idx;
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t x, int off) {
    const uint32_t lo = __shfl_xor((uint32_t)x, off), hi = __shfl_xor((uint32_t)(x >> 32), off);
    return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off);
    return x;
}

// A row in 16-byte vectors from its first aligned address: full vectors lo .. hi - 1,
// vector i holding entries i E - mis .., and at most 2 (E - 1) entries beside them.
template <typename T> struct Row {
    const T *p;
    int V, mis, lo, hi, head, tail0, tail;
    __device__ __forceinline__ Row(const T *row, int v) : p(row), V(v) {
        constexpr int E = Vec<T>::E;
        mis = (int)(((uintptr_t)row % 16) / sizeof(T));
        lo = mis ? 1 : 0;
        hi = (int)(((int64_t)V + mis) / E);
        head = mis ? min(E - mis, V) : 0;
        tail0 = max(hi, lo) * E - mis;
        tail = max(0, V - tail0);
    }
    __device__ __forceinline__ int first(int vec) const { return vec * Vec<T>::E - mis; }
    __device__ __forceinline__ uintx4 load(int vec) const {
        return *reinterpret_cast<const uintx4 *>(p + first(vec));
    }
    // the entry beside the full vectors that this thread looks after, or -1
    __device__ __forceinline__ int edge(int tid) const {
        return tid < head ? tid : tid < head + tail ? tail0 + tid - head : -1;
    }
    __device__ __forceinline__ float at(int i) const { return Elem<T>::load(p + i); }
};

// Any value of a row, slowly: k times the largest key below the one before.  For rows
// with NaN (which order above +inf) and for rows whose candidates overflow the list.
template <typename T, int THREADS>
__device__ __forceinline__ void top_by_passes(const Row<T> &row, int k, uint64_t *sKey, uint64_t *result) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    uint64_t prev = ~0ull;
    for (int r = 0; r < k; ++r) {
        uint64_t best = 0;
        for (int i = tid; i < row.V; i += THREADS) {
            const uint64_t key = make_key(row.at(i), i);
            if ((r == 0 || key < prev) && key > best) best = key;
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            const uint64_t o = shfl_xor64(best, off);
            best = o > best ? o : best;
        }
        __syncthreads();
        if (lane == 0) sKey[w] = best;
        __syncthreads();
        for (int v = 0; v < THREADS / 64; ++v) best = sKey[v] > best ? sKey[v] : best;
        if (tid == 0) result[r] = best;
        prev = best;
    }
    __syncthreads();
}

// Bound by HBM and, in bf16, nearly as much by the VALU (an exp, a maximum and five more
// operations an entry: 50 us of the 75).  4000 rows of 50261 bf16 (402 MB): 75 us without
// alternatives (5.3 TB/s), 82 with five, 86 with 32; 2048 rows fp32 (412 MB): 72 us (5.8 TB/s),
// 108 in a training pass, behind the 412 MB that the gradient before it has stored.  One
// row of 50261 fp32 with five alternatives: 10.5 us, the block's own latency.
template <typename T, int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS) row_kernel(Args a) {
    constexpr int E = Vec<T>::E, WAVES = THREADS / 64;
    constexpr int U = 32 / E;  // vectors of a batch: 32 entries, 64 or 128 bytes a thread in flight
    __shared__ float sM[WAVES], sS[WAVES], sT[WAVES];
    // the maxima of a thread's batches, SLOTS of them (batch i in slot i % SLOTS); the
    // listed candidates follow in the same memory
    constexpr int SLOTS = CAP * 2 / THREADS;
    __shared__ uint64_t sKey[TOP ? WAVES * 64 : 1], sCand[TOP ? CAP : 1], sTop[TOP ? MAX_K : 1];
    __shared__ uint64_t sBound;
    __shared__ int sCount, sOwners;
    __shared__ unsigned short sOwner[TOP ? SLOTS * THREADS : 1];  // slot * THREADS + thread
    float *sMax = reinterpret_cast<float *>(sCand);
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t n = blockIdx.x;
    const Row<T> row(static_cast<const T *>(a.logits) + n * a.ld, a.V);
    const float inv_t = 1.f / a.temperature, c = inv_t * LOG2E;
    const int64_t id = a.ids[n];
    const bool valid = id != a.ignore_index && id >= 0 && id < a.V;
    const float x_id = row.at(valid ? (int)id : 0);

    float m = -INFINITY, s = 0.f, t = 0.f;
    int batch_end = 0;  // the last entry of the batch that holds this thread's maximum
    auto add = [&](const float *x, int cnt, int last, int slot) {
        float bm = x[0];
#pragma unroll
        for (int i = 1; i < cnt; ++i) bm = fmaxf(bm, x[i]);
        if (TOP && slot >= 0) sMax[slot * THREADS + tid] = fmaxf(sMax[slot * THREADS + tid], bm);
        if (bm > m) {
            const float g = fmaxf((m - bm) * c, FLOOR), f = __builtin_amdgcn_exp2f(g);
            t = f * (t + s * g);
            s *= f;
            m = bm;
            batch_end = last;
        }
        const float mm = fmaxf(m, LOWEST);
#pragma unroll
        for (int i = 0; i < cnt; ++i) {
            const float u = (x[i] - mm) * c, e = __builtin_amdgcn_exp2f(u);
            s += e;
            t += e * fmaxf(u, FLOOR);
        }
    };
    if constexpr (TOP)
        for (int i = 0; i < SLOTS; ++i) sMax[i * THREADS + tid] = -INFINITY;
    int v0 = row.lo + tid, slot = 0;
    for (; v0 + (U - 1) * THREADS < row.hi; v0 += U * THREADS) {
        uintx4 r[U];
        float x[U * E];
#pragma unroll
        for (int i = 0; i < U; ++i) r[i] = row.load(v0 + i * THREADS);
#pragma unroll
        for (int i = 0; i < U; ++i) Vec<T>::unpack(r[i], x + i * E);
        add(x, U * E, row.first(v0 + (U - 1) * THREADS) + E - 1, slot);
        slot = (slot + 1) % SLOTS;
    }
    for (; v0 < row.hi; v0 += THREADS) {
        float x[E];
        Vec<T>::unpack(row.load(v0), x);
        add(x, E, row.first(v0) + E - 1, slot);
    }
    const int edge = row.edge(tid);
    if (edge >= 0) {
        const float x = row.at(edge);
        add(&x, 1, edge, -1);
    }

    // the block's maximum, s and t
    float M = wave_max(m);
    if (lane == 0) sM[w] = M;
    __syncthreads();
    M = sM[0];
    for (int v = 1; v < WAVES; ++v) M = fmaxf(M, sM[v]);
    {
        const float g = fmaxf((fmaxf(m, LOWEST) - fmaxf(M, LOWEST)) * c, FLOOR), f = __builtin_amdgcn_exp2f(g);
        t = wave_sum(f * (t + s * g));
        s = wave_sum(f * s);
    }
    if (lane == 0) {
        sS[w] = s;
        sT[w] = t;
    }
    if (TOP) {
        sKey[w * 64 + lane] = m > -INFINITY ? make_key(m, batch_end) : 0ull;
        if (tid == 0) sCount = sOwners = 0;
    }
    __syncthreads();
    s = t = 0.f;
    for (int v = 0; v < WAVES; ++v) {
        s += sS[v];
        t += sT[v];
    }
    const bool empty = s == 0.f;
    const float ln_s = logf(s);
    auto logprob = [&](float x) { return empty ? -INFINITY : (x - M) * inv_t - ln_s; };
    if (tid == 0) {
        a.logprobs[n] = valid ? logprob(x_id) : 0.f;
        a.entropy[n] = empty ? 0.f : ln_s - LN2 * (t / s);
        if (a.stats) {
            a.stats[2 * n] = M;
            a.stats[2 * n + 1] = s;
        }
    }
    if constexpr (TOP) {
        const int k = a.top_k;
        bool listed = s == s;  // NaN: by passes
        int count = 0;
        if (listed) {
            if (w == 0) {
                uint64_t mine = sKey[lane];
                for (int v = 1; v < WAVES; ++v) mine = sKey[v * 64 + lane] > mine ? sKey[v * 64 + lane] : mine;
                int above = 0;
                for (int i = 0; i < 64; ++i) {
                    const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), i) << 32) |
                                       (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
                    above += (o > mine || (o == mine && i < lane)) ? 1 : 0;
                }
                if (above == k - 1) sBound = mine;
            }
            __syncthreads();
            const uint64_t bound = sBound;  // 0: fewer than k groups hold anything
            auto list = [&](float x, int idx) {
                const uint64_t key = make_key(x, idx);
                if (x > -INFINITY && key >= bound) {
                    const int at = atomicAdd(&sCount, 1);
                    if (at < CAP) sCand[at] = key;
                }
            };
            const bool owner = m > -INFINITY && order(m) >= (uint32_t)(bound >> 32);
            if (owner)
                for (int i = 0; i < SLOTS; ++i) {
                    const float x = sMax[i * THREADS + tid];
                    if (x > -INFINITY && order(x) >= (uint32_t)(bound >> 32))
                        sOwner[atomicAdd(&sOwners, 1)] = (unsigned short)(i * THREADS + tid);
                }
            __syncthreads();
            if (owner && edge >= 0) list(row.at(edge), edge);
            // (owner's slot, its j-th vector) over the block's threads
            const int batches = (row.hi - row.lo + U * THREADS - 1) / (U * THREADS);
            const int per = (batches + SLOTS - 1) / SLOTS * U, total = sOwners * per;
            for (int i = tid; i < total; i += THREADS) {
                const int o = i / per, j = i - o * per, code = sOwner[o];
                const int vec = (j / U * SLOTS + code / THREADS) * U + j % U;
                const int64_t v = row.lo + code % THREADS + (int64_t)vec * THREADS;
                if (v >= row.hi) continue;
                float x[E];
                Vec<T>::unpack(row.load((int)v), x);
#pragma unroll
                for (int e = 0; e < E; ++e) list(x[e], row.first((int)v) + e);
            }
            __syncthreads();
            count = sCount;
            listed = count <= CAP;
        }
        if (listed) {
            for (int i = tid; i < count; i += THREADS) {
                const uint64_t mine = sCand[i];
                int above = 0;
                for (int j = 0; j < count; ++j) above += sCand[j] > mine ? 1 : 0;
                if (above < k) sTop[above] = mine;
            }
            // fewer than k entries above -inf: the masked ones of lowest index, all below k
            if (count < k && w == 0) {
                const bool masked = lane < k && row.at(lane < k ? lane : 0) == -INFINITY;
                const uint64_t b = __ballot(masked);
                const int at = count + __popcll(b & ((1ull << lane) - 1));
                if (masked && at < k) sTop[at] = make_key(-INFINITY, lane);
            }
            __syncthreads();
        } else {
            top_by_passes<T, THREADS>(row, k, sKey, sTop);
        }
        if (tid < k) {
            const uint64_t key = sTop[tid];
            a.top_ids[n * k + tid] = (int64_t)(uint32_t)~(uint32_t)key;
            a.top_logprobs[n * k + tid] = logprob(unorder((uint32_t)(key >> 32)));
        }
    }
}

// -------------------------------------------------------------- gradient ---
constexpr int GT = 256, GV = 8;  // threads, vectors per thread and block

template <typename T> __device__ __forceinline__ uintx4 pack(const float *x);
template <> __device__ __forceinline__ uintx4 pack<float>(const float *x) {
    return uintx4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
}
template <> __device__ __forceinline__ uintx4 pack<unsigned short>(const float *x) {
    return uintx4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}
__device__ __forceinline__ void put(float *p, float x) { *p = x; }
__device__ __forceinline__ void put(unsigned short *p, float x) { *p = __builtin_bit_cast(unsigned short, (__bf16)x); }

// A block writes a stretch of one row's gradient without the terms of the given and
// top tokens, then overwrites those entries that fall into its stretch.  VECTORS: the
// row of logits and the row of the gradient start at the same offset from 16 bytes.
// Bound by HBM: 2048 rows of 50261 fp32, 412 MB read and as much written, 141 us (5.8 TB/s).
template <typename T, bool VECTORS>
__global__ void __launch_bounds__(GT) grad_kernel(Args a, int segs) {
    constexpr int E = Vec<T>::E;
    const int tid = threadIdx.x;
    const int64_t n = blockIdx.x / (unsigned)segs;
    const int seg = (int)(blockIdx.x - n * segs);
    const Row<T> row(static_cast<const T *>(a.logits) + n * a.ld, a.V);
    T *out = static_cast<T *>(a.d_logits) + n * a.ldd;
    const int64_t id = a.ids[n];
    const bool valid = id != a.ignore_index && id >= 0 && id < a.V;
    const float inv_t = 1.f / a.temperature, c = inv_t * LOG2E;
    const float M = a.stats[2 * n], s = a.stats[2 * n + 1], inv_s = s == 0.f ? 0.f : 1.f / s;
    const float g_lp = valid && a.g_logprobs ? a.g_logprobs[n] : 0.f;
    const float g_ent = a.g_entropy ? a.g_entropy[n] : 0.f;
    float g_all = g_lp;
    if (a.g_top)
        for (int i = 0; i < a.top_k; ++i) g_all += a.g_top[n * a.top_k + i];
    // ln p_v + entropy = ln2 u_v + (entropy - ln s)
    const float base = g_all + g_ent * (a.entropy[n] - logf(s)), slope = g_ent * LN2;
    const float mm = fmaxf(M, LOWEST), k = -inv_t * inv_s;
    auto value = [&](float x, float extra) {
        if (s == 0.f) return 0.f;
        const float u = (x - mm) * c;
        return k * __builtin_amdgcn_exp2f(u) * (base + slope * fmaxf(u, FLOOR)) + inv_t * extra;
    };
    int e0, e1;  // this block's entries
    if constexpr (VECTORS) {
        const int b0 = row.lo + seg * GT * GV, b1 = min(row.hi, b0 + GT * GV);
#pragma unroll 4
        for (int v = b0 + tid; v < b1; v += GT) {
            float x[E];
            Vec<T>::unpack(row.load(v), x);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = value(x[i], 0.f);
            *reinterpret_cast<uintx4 *>(out + row.first(v)) = pack<T>(x);
        }
        e0 = seg == 0 ? 0 : row.first(b0);
        e1 = seg == segs - 1 ? a.V : row.first(b0 + GT * GV);
        const int edge = row.edge(tid);
        if (edge >= e0 && edge < e1) put(out + edge, value(row.at(edge), 0.f));
    } else {
        e0 = seg * GT * GV * E;
        e1 = min(a.V, e0 + GT * GV * E);
        for (int i = e0 + tid; i < e1; i += GT) put(out + i, value(row.at(i), 0.f));
    }
    __syncthreads();  // the stretch is written
    const int special = a.g_top ? a.top_k + 1 : 1;
    if (tid < special) {
        const bool token = tid == special - 1;
        const int64_t v = token ? (valid ? id : -1) : a.top_ids[n * a.top_k + tid];
        if (v < e0 || v >= e1) return;
        float extra = 0.f;
        if (a.g_top)
            for (int i = 0; i < a.top_k; ++i)
                if (a.top_ids[n * a.top_k + i] == v) extra += a.g_top[n * a.top_k + i];
        if (valid && v == id) extra += g_lp;
        put(out + v, value(row.at((int)v), extra));
    }
}

int check(const Args &a, const char *who) {
    QPAM_REQUIRE(a.dtype == QPAM_F32 || a.dtype == QPAM_BF16, "%s: dtype %d", who, a.dtype);
    QPAM_REQUIRE(a.n >= 0 && a.n < (1ll << 31) && a.V >= 1 && a.V <= (1 << 30), "%s: bad sizes n=%lld V=%d", who,
                 (long long)a.n, a.V);
    QPAM_REQUIRE(a.temperature >= 1e-30f && a.temperature <= 1e30f, "%s: temperature %g outside 1e-30 .. 1e30", who,
                 a.temperature);
    QPAM_REQUIRE(a.top_k >= 0 && a.top_k <= MAX_K && a.top_k <= a.V, "%s: top_k %d (0 to %d, at most V=%d)", who, a.top_k,
                 MAX_K, a.V);
    QPAM_REQUIRE(a.n == 0 || (a.logits && a.ids && a.entropy && a.ld >= a.V), "%s: null pointer or row stride below V", who);
    QPAM_REQUIRE((uintptr_t)a.logits % (a.dtype == QPAM_F32 ? 4 : 2) == 0, "%s: logits not aligned to their type", who);
    return QPAM_OK;
}

// A launch holds less than 2^32 threads: more blocks of 256 go in several.
constexpr int64_t MAX_BLOCKS = (int64_t)1 << 23;

// rows n0 .. n0 + n - 1 of a call
template <typename T> Args rows_of(Args a, int64_t n0, int64_t n) {
    auto move = [](auto *&p, int64_t by) {
        if (p) p += by;
    };
    a.n = n;
    a.logits = static_cast<const T *>(a.logits) + n0 * a.ld;
    if (a.d_logits) a.d_logits = static_cast<T *>(a.d_logits) + n0 * a.ldd;
    move(a.ids, n0);
    move(a.logprobs, n0);
    move(a.entropy, n0);
    move(a.stats, 2 * n0);
    move(a.top_logprobs, n0 * a.top_k);
    move(a.top_ids, n0 * a.top_k);
    move(a.g_logprobs, n0);
    move(a.g_entropy, n0);
    move(a.g_top, n0 * a.top_k);
    return a;
}

template <typename T, int THREADS>
int launch_rows(const Args &a, hipStream_t stream) {
    if (a.top_k)
        hipLaunchKernelGGL((row_kernel<T, THREADS, true>), dim3((unsigned)a.n), dim3(THREADS), 0, stream, a);
    else
        hipLaunchKernelGGL((row_kernel<T, THREADS, false>), dim3((unsigned)a.n), dim3(THREADS), 0, stream, a);
    return launch_status("logprobs row_kernel");
}

// Up to 256 long rows, one a CU: 1024 threads a block (192 rows of 50261 fp32: 12.8 us
// against 21).  More rows fill the CUs with blocks of 256 (512 rows: 21.0 us against 21.9
// with 1024 threads, with five alternatives 25.1 against 32.0).
template <typename T>
int run_rows(const Args &a, hipStream_t stream) {
    if (a.n <= 256 && a.V >= 16384) return launch_rows<T, 1024>(a, stream);
    for (int64_t n0 = 0; n0 < a.n; n0 += MAX_BLOCKS) {
        const int st = launch_rows<T, 256>(rows_of<T>(a, n0, std::min(MAX_BLOCKS, a.n - n0)), stream);
        if (st) return st;
    }
    return QPAM_OK;
}

template <typename T>
int run_grad(const Args &a, hipStream_t stream) {
    constexpr int64_t STRETCH = (int64_t)GT * GV * Vec<T>::E;
    const int segs = (int)((a.V + STRETCH - 1) / STRETCH);
    const int64_t per = std::max<int64_t>(1, MAX_BLOCKS / segs);  // rows of a launch
    const bool vectors = (uintptr_t)a.logits % 16 == (uintptr_t)a.d_logits % 16 &&
                         (a.n == 1 || (a.ld - a.ldd) * (int64_t)sizeof(T) % 16 == 0);
    for (int64_t n0 = 0; n0 < a.n; n0 += per) {
        const Args s = rows_of<T>(a, n0, std::min(per, a.n - n0));
        if (vectors)
            hipLaunchKernelGGL((grad_kernel<T, true>), dim3((unsigned)(s.n * segs)), dim3(GT), 0, stream, s, segs);
        else
            hipLaunchKernelGGL((grad_kernel<T, false>), dim3((unsigned)(s.n * segs)), dim3(GT), 0, stream, s, segs);
        const int st = launch_status("logprobs grad_kernel");
        if (st) return st;
    }
    return QPAM_OK;
}

}  // namespace
}  // namespace logprobs
}  // namespace qpam

extern "C" int qpam_logprobs_fwd(const qpam_logprobs_args *a, void *stream) {
    using namespace qpam;
    using namespace qpam::logprobs;
    QPAM_REQUIRE(a != nullptr, "qpam_logprobs_fwd: null args");
    int st = check(*a, "qpam_logprobs_fwd");
    if (st || a->n == 0) return st;
    QPAM_REQUIRE(a->logprobs && (a->top_k == 0 || (a->top_logprobs && a->top_ids)), "qpam_logprobs_fwd: null output");
    return a->dtype == QPAM_BF16 ? run_rows<unsigned short>(*a, (hipStream_t)stream)
                                 : run_rows<float>(*a, (hipStream_t)stream);
}

extern "C" int qpam_logprobs_bwd(const qpam_logprobs_args *a, void *stream) {
    using namespace qpam;
    using namespace qpam::logprobs;
    QPAM_REQUIRE(a != nullptr, "qpam_logprobs_bwd: null args");
    int st = check(*a, "qpam_logprobs_bwd");
    if (st || a->n == 0) return st;
    QPAM_REQUIRE(a->stats && a->d_logits && a->ldd >= a->V, "qpam_logprobs_bwd: null stats or d_logits, or row stride below V");
    QPAM_REQUIRE(!a->g_top || (a->top_k && a->top_ids), "qpam_logprobs_bwd: g_top without top_ids");
    QPAM_REQUIRE((uintptr_t)a->d_logits % (a->dtype == QPAM_F32 ? 4 : 2) == 0, "qpam_logprobs_bwd: d_logits not aligned to its type");
    return a->dtype == QPAM_BF16 ? run_grad<unsigned short>(*a, (hipStream_t)stream)
                                 : run_grad<float>(*a, (hipStream_t)stream);
}
