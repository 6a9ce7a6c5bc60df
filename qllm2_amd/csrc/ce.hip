// Tied complex LM-head cross-entropy (fused GEMM + softmax statistics).
//
// Reference: _FusedLinearCE (v11/fused_ce.py:26-82), linear_ce_per_token and
// linear_ce_stats (v11/fused_ce.py:98-141), called from V11LM.ce_from_lm
// (v11/model.py:1175-1190) with H = [lm_r | lm_i], W = [E_r | E_i] so that
// H W^T = Re(h conj(E)^T).
//
// Forward: one MFMA GEMM tile per (rows, vocab) block (256 x 128 for bf16,
// 128 x 128 for fp32) whose epilogue reduces the tile to per-row (max, sum exp,
// argmax); logits never leave registers.  A per-row finalize merges the vocab
// tiles into lse, adds the target logit (a direct dot product) and writes the
// per-row loss; a single-block reduction produces the loss sum and the
// denominator.
// Backward, per `chunk` rows: the same GEMM recomputes the logits tile and its
// epilogue writes G = (softmax - onehot) * scale in the input dtype as
// G^T [vocab][rows] (and G [rows][vocab] where a hand-written GEMM reads it);
// then the two plain GEMMs dW += G^T H and dH = G W run through hipBLASLt
// (bf16, blas.hip) or through the hand-written K-contiguous GEMM kernels (W^T
// and H^T transposed once into the workspace).  The G buffers hold `chunk`
// rows, the reference's own memory bound (it keeps chunk x V fp32 logits and
// softmax alive).
//
// Token scores (qpam_linear_logprobs_*; namespaces split for fp32, tiles for bf16, thin
// for few rows, with products of their own): the log probability of each row's token and
// the entropy of the row.  With c = log2(e) / T, m = max x and u = c (x - m), the tiles
// reduce s = sum 2^u and t = sum 2^u u, so that
//   log prob = ln2 (u_token - log2 s),   entropy = ln2 (log2 s - t / s),
// with the token's logit from the same accumulators (the tile that holds its column keeps it),
// and the gradient tiles write (as G^T alone)
//   G_v = -p_v / T (g_lp + g_ent (ln p_v + entropy)) + [v = token] g_lp / T.
// The maximum is taken off in front of c: a reference of c m in fp32 is off by 2^-25 of
// itself, which is past the exponent's range from |c m| = 2^32 on (T = 1e-9).
#include <algorithm>
#include <type_traits>

#include "blas.h"
#include "common.h"

namespace qpam {
namespace ce {
namespace {

constexpr int THREADS = 256;
constexpr int BM = 128, BN = 128, BK = 32;
constexpr int VT = 128;  // vocab tile

template <typename T> struct Mma;

// bf16 inputs: v_mfma_f32_16x16x32_bf16, lane supplies 8 consecutive k
template <> struct Mma<unsigned short> {
    static constexpr int PITCH = BK + 8;  // elements per LDS row (80 bytes)
    static constexpr int ROW16 = BK * 2 / 16;  // 16-byte chunks per tile row
    __device__ __forceinline__ static void step(const unsigned short *sA, const unsigned short *sB, int arow0,
                                                int brow0, floatx4 (&acc)[4][4], int l16, int g) {
        bf16x8 af[4], bfr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            af[i] = *reinterpret_cast<const bf16x8 *>(sA + (arow0 + 16 * i + l16) * PITCH + 8 * g);
            bfr[i] = *reinterpret_cast<const bf16x8 *>(sB + (brow0 + 16 * i + l16) * PITCH + 8 * g);
        }
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
#pragma unroll
            for (int ni = 0; ni < 4; ++ni)
                acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[mi], bfr[ni], acc[mi][ni], 0, 0, 0);
    }
};

// fp32 inputs: v_mfma_f32_16x16x4_f32, k-steps use k = 16q + 4g + kk
template <> struct Mma<float> {
    static constexpr int PITCH = BK + 4;
    static constexpr int ROW16 = BK * 4 / 16;
    __device__ __forceinline__ static void step(const float *sA, const float *sB, int arow0, int brow0,
                                                floatx4 (&acc)[4][4], int l16, int g) {
#pragma unroll
        for (int q = 0; q < BK / 16; ++q) {
            float4 af[4], bfr[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                af[i] = *reinterpret_cast<const float4 *>(sA + (arow0 + 16 * i + l16) * PITCH + 16 * q + 4 * g);
                bfr[i] = *reinterpret_cast<const float4 *>(sB + (brow0 + 16 * i + l16) * PITCH + 16 * q + 4 * g);
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
#pragma unroll
                for (int mi = 0; mi < 4; ++mi)
#pragma unroll
                    for (int ni = 0; ni < 4; ++ni)
                        acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x4f32(af[mi][kk], bfr[ni][kk], acc[mi][ni], 0,
                                                                           0, 0);
        }
    }
};

template <typename T>
constexpr size_t gemm_smem() { return (size_t)2 * (BM + BN) * Mma<T>::PITCH * sizeof(T); }

// C[m][n] = sum_k A[m][k] B[n][k] for one BM x BN tile; A and B point at the
// tile's first row; rows beyond a_rows / b_rows read as zero; K % BK == 0.
// Wave w owns rows 64*(w>>1).., cols 64*(w&1)..; acc[mi][ni] lane holds
// C[64*(w>>1) + 16mi + 4g + r][64*(w&1) + 16ni + l16].
template <typename T>
__device__ __forceinline__ void gemm_tile(const T *A, int64_t lda, int a_rows, const T *B, int64_t ldb, int b_rows,
                                          int K, floatx4 (&acc)[4][4], T *smem) {
    using MM = Mma<T>;
    constexpr int PITCH = MM::PITCH, R16 = MM::ROW16, EPC = 16 / sizeof(T);
    constexpr int LOADS = BM * R16 / THREADS;  // 16-byte loads per thread per operand
    // buffers by offset: a table of pointers loses their address space, and flat loads
    // from LDS wait for the global loads in flight as well
    auto sA = [&](int buf) { return smem + buf * (BM + BN) * PITCH; };
    auto sB = [&](int buf) { return smem + (buf * (BM + BN) + BM) * PITCH; };
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int arow0 = 64 * (w >> 1), brow0 = 64 * (w & 1);
#pragma unroll
    for (int mi = 0; mi < 4; ++mi)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = floatx4{0.f, 0.f, 0.f, 0.f};

    uint4 ra[LOADS], rb[LOADS];
    auto gload = [&](int k0) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int ci = tid + i * THREADS, row = ci / R16, c = ci % R16;
            ra[i] = (row < a_rows) ? *reinterpret_cast<const uint4 *>(A + row * lda + k0 + c * EPC)
                                   : make_uint4(0, 0, 0, 0);
            rb[i] = (row < b_rows) ? *reinterpret_cast<const uint4 *>(B + row * ldb + k0 + c * EPC)
                                   : make_uint4(0, 0, 0, 0);
        }
    };
    auto lstore = [&](int buf) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int ci = tid + i * THREADS, row = ci / R16, c = ci % R16;
            *reinterpret_cast<uint4 *>(sA(buf) + row * PITCH + c * EPC) = ra[i];
            *reinterpret_cast<uint4 *>(sB(buf) + row * PITCH + c * EPC) = rb[i];
        }
    };
    const int KT = K / BK;
    gload(0);
    lstore(0);
    __syncthreads();
    for (int kt = 0; kt < KT; ++kt) {
        const int buf = kt & 1;
        if (kt + 1 < KT) gload((kt + 1) * BK);
        MM::step(sA(buf), sB(buf), arow0, brow0, acc, l16, g);
        if (kt + 1 < KT) lstore(buf ^ 1);
        __syncthreads();
    }
}

// ------------------------------------------------------------ forward -----
constexpr float LN2 = 0.6931471805599453f, LOG2 = 1.4426950408889634f;
constexpr float U_FLOOR = -1e4f;  // 2^u is 0 and 2^u u is -0, not NaN

struct FwdParams {
    qpam_ce_fwd_args a;
    int n_vt;
    float *part_m, *part_s;  // [N][n_vt]
    int *part_i;             // [N][n_vt] argmax
    float *red;              // [2] loss sum, denominator
    // token scores
    float *part_t;           // [N][n_vt] sum of 2^u u, in part_i's place
    int full_vt;             // vocab tiles of 256 columns in front of the narrow ones (tiles::Columns)
    float c;                 // log2(e) / T
    float *token_x;          // [N] the logit of the row's token, as the tiles' sums have it
    float *logprobs, *entropy, *stats;
};

// the row's token, or -1: none, or no such row
__device__ __forceinline__ int token_of(const FwdParams &p, int64_t id) {
    return id != p.a.ignore_index && id >= 0 && id < p.a.V ? (int)id : -1;
}
__device__ __forceinline__ int row_token(const FwdParams &p, int row) { return row < p.a.N ? token_of(p, p.a.targets[row]) : -1; }

// A lane's logits of one row, in columns v, v + 16, ..: the token's, if it is one of them, is
// what the row's maximum and sums hold, so its log probability is at most 0.
template <int NI> __device__ __forceinline__ void keep_token(const FwdParams &p, const floatx4 (&x)[NI], int r, int row, int token, int v) {
    const unsigned at = (unsigned)(token - v);  // past 2^31 where there is none
    if (at < 16u * NI && at % 16 == 0) {
        float y = x[0][r];
#pragma unroll
        for (int ni = 1; ni < NI; ++ni) y = at == 16u * ni ? x[ni][r] : y;
        p.token_x[row] = y;
    }
}

// (m, s, t) of two parts of a row's logits as one (m = -inf: a part of nothing)
__device__ __forceinline__ void join_scores(float c, float &m, float &s, float &t, float om, float os, float ot) {
    const float nm = fmaxf(m, om), lo = fmaxf(nm, -3.402823466e38f);
    const float g = fmaxf((m - lo) * c, U_FLOOR), og = fmaxf((om - lo) * c, U_FLOOR);
    const float f = __builtin_amdgcn_exp2f(g), of = __builtin_amdgcn_exp2f(og);
    t = f * (t + s * g) + of * (ot + os * og);
    s = f * s + of * os;
    m = nm;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) ce_fwd_tile_kernel(FwdParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T *smem = reinterpret_cast<T *>(smem_raw);
    __shared__ float sM[2][BM], sS[2][BM];
    __shared__ int sI[2][BM];
    const qpam_ce_fwd_args &a = p.a;
    const int vt = blockIdx.x, rt = blockIdx.y;
    const int r0 = rt * BM, v0 = vt * VT;
    floatx4 acc[4][4];
    gemm_tile<T>((const T *)a.h + (int64_t)r0 * a.ldh, a.ldh, min(BM, a.N - r0), (const T *)a.w + (int64_t)v0 * a.ldw,
                 a.ldw, min(BN, a.V - v0), a.D, acc, smem);

    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
#pragma unroll
    for (int mi = 0; mi < 4; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float mx = -INFINITY;
            int ix = 0x7fffffff;
#pragma unroll
            for (int ni = 0; ni < 4; ++ni) {
                const int v = v0 + 64 * wn + 16 * ni + l16;
                const float x = (v < a.V) ? acc[mi][ni][r] : -INFINITY;
                if (x > mx) { mx = x; ix = v; }
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) {
                const float om = __shfl_xor(mx, off);
                const int oi = __shfl_xor(ix, off);
                if (om > mx || (om == mx && oi < ix)) { mx = om; ix = oi; }
            }
            float s = 0.f;
#pragma unroll
            for (int ni = 0; ni < 4; ++ni) {
                const int v = v0 + 64 * wn + 16 * ni + l16;
                if (v < a.V) s += __expf(acc[mi][ni][r] - mx);
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) s += __shfl_xor(s, off);
            if (l16 == 0) {
                const int row = 64 * wm + 16 * mi + 4 * g + r;
                sM[wn][row] = mx;
                sS[wn][row] = s;
                sI[wn][row] = ix;
            }
        }
    }
    __syncthreads();
    if (tid < BM && r0 + tid < a.N) {
        const float m0 = sM[0][tid], m1 = sM[1][tid];
        const float m = fmaxf(m0, m1);
        float s = 0.f;
        if (m0 > -INFINITY) s += sS[0][tid] * __expf(m0 - m);
        if (m1 > -INFINITY) s += sS[1][tid] * __expf(m1 - m);
        const int i = (m1 > m0 || (m1 == m0 && sI[1][tid] < sI[0][tid])) ? sI[1][tid] : sI[0][tid];
        const int64_t o = (int64_t)(r0 + tid) * p.n_vt + vt;
        p.part_m[o] = m;
        p.part_s[o] = s;
        p.part_i[o] = i;
    }
}

// one wave per row: merge the vocab tiles, add the target logit
template <typename T>
__global__ void __launch_bounds__(THREADS) ce_fwd_finalize_kernel(FwdParams p) {
    const qpam_ce_fwd_args &a = p.a;
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6);
    if (row >= a.N) return;
    float m = -INFINITY, s = 0.f;
    int ix = 0x7fffffff;
    for (int vt = lane; vt < p.n_vt; vt += 64) {
        const int64_t o = (int64_t)row * p.n_vt + vt;
        const float pm = p.part_m[o], ps = p.part_s[o];
        const int pi = a.correct ? p.part_i[o] : 0;  // tile argmax, written only when requested
        if (pm > m || (pm == m && pi < ix)) ix = pi;
        const float nm = fmaxf(m, pm);
        s = (m > -INFINITY ? s * __expf(m - nm) : 0.f) + (pm > -INFINITY ? ps * __expf(pm - nm) : 0.f);
        m = nm;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const float om = __shfl_xor(m, off), os = __shfl_xor(s, off);
        const int oi = __shfl_xor(ix, off);
        const float nm = fmaxf(m, om);
        const float ns = (m > -INFINITY ? s * __expf(m - nm) : 0.f) + (om > -INFINITY ? os * __expf(om - nm) : 0.f);
        if (om > m || (om == m && oi < ix)) ix = oi;
        m = nm;
        s = ns;
    }
    const float lse = m + __logf(s);
    const int64_t t = a.targets[row];
    const bool valid = (t != a.ignore_index) && t >= 0 && t < a.V;
    float dot = 0.f;
    if (valid) {
        const T *hr = (const T *)a.h + (int64_t)row * a.ldh;
        const T *wr = (const T *)a.w + t * a.ldw;
        for (int k = lane; k < a.D; k += 64) dot += Elem<T>::load(hr + k) * Elem<T>::load(wr + k);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) dot += __shfl_xor(dot, off);
    if (lane == 0) {
        float loss = valid ? (lse - dot) : 0.f;
        if (a.mask) loss *= a.mask[row];
        a.lse[row] = lse;
        a.loss[row] = loss;
        if (a.correct) a.correct[row] = (valid && ix == t) ? 1.f : 0.f;
    }
}

// one wave per row: merge the vocab tiles into (m, s, t), add the token's logit.  Neither
// a log probability above 0 nor an entropy below it is left by the last roundings.
__global__ void __launch_bounds__(THREADS) scores_finalize_kernel(FwdParams p) {
    const qpam_ce_fwd_args &a = p.a;
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * (THREADS / 64) + (threadIdx.x >> 6);
    if (row >= a.N) return;
    float m = -INFINITY, s = 0.f, t = 0.f;
    for (int vt = lane; vt < p.n_vt; vt += 64) {
        const int64_t o = (int64_t)row * p.n_vt + vt;
        join_scores(p.c, m, s, t, p.part_m[o], p.part_s[o], p.part_t[o]);
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1)
        join_scores(p.c, m, s, t, __shfl_xor(m, off), __shfl_xor(s, off), __shfl_xor(t, off));
    if (lane == 0) {
        const float log_s = log2f(s), ent = LN2 * (log_s - t / s);
        float lp = 0.f;
        if (row_token(p, row) >= 0) lp = LN2 * ((p.token_x[row] - m) * p.c - log_s);
        p.logprobs[row] = lp > 0.f ? 0.f : lp;
        p.entropy[row] = ent < 0.f ? 0.f : ent;
        p.stats[2 * row] = m;
        p.stats[2 * row + 1] = s;
    }
}

// deterministic single-block sum: red[0] = sum loss, red[1] = denominator
__global__ void __launch_bounds__(1024) ce_reduce_kernel(FwdParams p) {
    const qpam_ce_fwd_args &a = p.a;
    __shared__ float s1[32], s2[32];
    float x = 0.f, y = 0.f;
    for (int r = threadIdx.x; r < a.N; r += 1024) {
        x += a.loss[r];
        if (a.mask) {
            y += a.mask[r];
        } else {
            const int64_t t = a.targets[r];
            y += (t != a.ignore_index) ? 1.f : 0.f;
        }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        x += __shfl_xor(x, off);
        y += __shfl_xor(y, off);
    }
    if ((threadIdx.x & 63) == 0) {
        s1[threadIdx.x >> 6] = x;
        s2[threadIdx.x >> 6] = y;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float tx = 0.f, ty = 0.f;
        for (int i = 0; i < 16; ++i) {
            tx += s1[i];
            ty += s2[i];
        }
        a.loss_sum[0] = tx;
        a.loss_sum[1] = ty;
    }
}

// ----------------------------------------------------------- backward -----
struct BwdParams {
    qpam_ce_bwd_args a;
    int Vp;          // vocab padded to VT
    int Rp;          // chunk rows padded to BK
    int row0;        // first row of the chunk
    int rows;        // rows in the chunk
    void *wt;        // [D][Vp]
    void *gbuf;      // [rows][Vp]
    void *gtbuf;     // [Vp][Rp]
    void *ht;        // [D][Rp]
    int write_g;     // bf16 path: also write G (only the hand-written dH GEMM reads it)
    // token scores
    int full_vt;     // vocab tiles of 256 columns in front of the narrow ones (tiles::Columns)
    float inv_t, c;  // 1 / T, log2(e) / T
    const float *stats, *logprobs, *entropy, *g_logprobs, *g_entropy;
    // bf16: G at the rows' tokens, in fp32 and not in G^T (scores_token_kernel); room for Rp rows
    float *token_g;
    int *token_id;  // -1: no token
};

// A row's part of G_v = 2^u (base + slope u), u = c (x - m).  Zero for a row past the end.
struct RowScore {
    float m, base, slope;
};

// u of one logit, kept where 2^u (base + slope u) is finite: above U_FLOOR, past which 2^u is 0
// but slope u can be infinite (low temperatures), and at most 0, as the maximum is the
// forward's and this sum may be off from it in its last bits.  A row with NaN has a NaN base.
__device__ __forceinline__ float score_u(float x, float m, float c) { return __builtin_amdgcn_fmed3f((x - m) * c, U_FLOOR, 0.f); }

__device__ __forceinline__ RowScore row_score(const BwdParams &p, int lr) {
    if (lr >= p.rows) return {0.f, 0.f, 0.f};
    const qpam_ce_bwd_args &a = p.a;
    const int row = p.row0 + lr;
    const int64_t id = a.targets[row];
    const bool valid = id != a.ignore_index && id >= 0 && id < a.V;
    const float s = p.stats[2 * row + 1], k = -p.inv_t / s;
    const float g_lp = valid && p.g_logprobs ? p.g_logprobs[row] : 0.f, g_ent = p.g_entropy ? p.g_entropy[row] : 0.f;
    return {p.stats[2 * row], k * (g_lp + g_ent * (p.entropy[row] - LN2 * log2f(s))), k * g_ent * LN2};
}

// G at the rows' tokens, where the tiles left out the one-hot term: with p = e^logprob
//   G = (g_lp (1 - p) - g_ent p (logprob + entropy)) / T,
// in fp32 to G^T.  In bf16 it stays out of G^T (0 there) and joins the products' sums in fp32
// (tiles::gemm_kernel): it is the largest entry of most rows, and its rounding to bf16 was nearly
// all of the gradients' error beyond that of their own rounding (16384 x 50261 x 1024: 2.4e-3
// with it, 1.7e-3 without, as products of an fp32 G).  The other entries are rounded to bf16,
// 2^-8 of each at most and so little of the row where p is spread; G in two bf16 parts would
// double the work of both products (2.7 of 6.1 ms).
template <typename T>
__global__ void __launch_bounds__(THREADS) scores_token_kernel(BwdParams p) {
    const qpam_ce_bwd_args &a = p.a;
    const int lr = blockIdx.x * THREADS + threadIdx.x, row = p.row0 + lr;
    if (lr >= p.rows) return;
    const int64_t id = a.targets[row];
    const bool valid = id != a.ignore_index && id >= 0 && id < a.V;
    if (sizeof(T) == 2) p.token_id[lr] = valid ? (int)id : -1;
    if (!valid) return;
    const float g_lp = p.g_logprobs ? p.g_logprobs[row] : 0.f, g_ent = p.g_entropy ? p.g_entropy[row] : 0.f;
    const float lp = p.logprobs[row], q = expf(lp);
    const float x = p.inv_t * (g_lp * (1.f - q) - g_ent * q * (fmaxf(lp, U_FLOOR) + p.entropy[row]));
    if (sizeof(T) == 2) p.token_g[lr] = x;
    static_cast<T *>(p.gtbuf)[id * p.Rp + lr] = sizeof(T) == 2 ? T(0) : T(x);
}

// out[c][r] = in[r][c] for an R x Cc tile grid (64 x 64 LDS tiles); rows >= R
// and cols >= Cc of the (padded) output are written as zero.
template <typename T>
__global__ void __launch_bounds__(THREADS) transpose_kernel(const T *in, int64_t ldi, int R, int Cc, T *out,
                                                           int64_t ldo, int out_rows, int out_cols) {
    __shared__ T tile[64][65];
    const int c0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
    for (int e = threadIdx.x; e < 64 * 64; e += THREADS) {
        const int rr = e >> 6, cc = e & 63;
        const int r = r0 + rr, c = c0 + cc;
        tile[rr][cc] = (r < R && c < Cc) ? in[(int64_t)r * ldi + c] : T(0);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 64 * 64; e += THREADS) {
        const int cc = e >> 6, rr = e & 63;
        const int orow = c0 + cc, ocol = r0 + rr;
        if (orow < out_rows && ocol < out_cols) out[(int64_t)orow * ldo + ocol] = tile[rr][cc];
    }
}

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ unsigned short from_f32<unsigned short>(float x) { return f32_to_bf16(x); }

// G tile: recompute logits, G = (exp(x - lse) - [v == t]) * scale; write G and G^T
template <typename T>
__global__ void __launch_bounds__(THREADS) ce_grad_tile_kernel(BwdParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T *smem = reinterpret_cast<T *>(smem_raw);
    __shared__ float sLse[BM], sScale[BM];
    __shared__ int sTgt[BM];
    const qpam_ce_bwd_args &a = p.a;
    const int vt = blockIdx.x, rt = blockIdx.y;
    const int lr0 = rt * BM, v0 = vt * VT;          // chunk-local row
    const int tid = threadIdx.x;
    if (tid < BM) {
        const int lr = lr0 + tid, row = p.row0 + lr;
        float lse = 0.f, sc = 0.f;
        int tg = -1;
        if (lr < p.rows) {
            const int64_t t = a.targets[row];
            const bool valid = (t != a.ignore_index) && t >= 0 && t < a.V;
            lse = a.lse[row];
            sc = valid ? a.grad_scale[0] * (a.mask ? a.mask[row] : 1.f) : 0.f;
            tg = valid ? (int)t : -1;
        }
        sLse[tid] = lse;
        sScale[tid] = sc;
        sTgt[tid] = tg;
    }
    floatx4 acc[4][4];
    gemm_tile<T>((const T *)a.h + (int64_t)(p.row0 + lr0) * a.ldh, a.ldh, min(BM, p.rows - lr0),
                 (const T *)a.w + (int64_t)v0 * a.ldw, a.ldw, min(BN, a.V - v0), a.D, acc, smem);
    const int w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
    T *G = (T *)p.gbuf;
    T *GT = (T *)p.gtbuf;
#pragma unroll
    for (int mi = 0; mi < 4; ++mi) {
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) {
            const int vloc = 64 * wn + 16 * ni + l16, v = v0 + vloc;
            T gv[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int rl = 64 * wm + 16 * mi + 4 * g + r;
                float x = 0.f;
                if (v < a.V && sScale[rl] != 0.f) {
                    x = __expf(acc[mi][ni][r] - sLse[rl]);
                    if (v == sTgt[rl]) x -= 1.f;
                    x *= sScale[rl];
                }
                gv[r] = from_f32<T>(x);
                const int lr = lr0 + rl;
                if (lr < p.rows) G[(int64_t)lr * p.Vp + v] = gv[r];
            }
            // G^T[v][lr0 + 64wm + 16mi + 4g .. +3]: 4 consecutive rows
            T *dst = GT + (int64_t)v * p.Rp + lr0 + 64 * wm + 16 * mi + 4 * g;
            if (lr0 + 64 * wm + 16 * mi + 4 * g + 3 < p.Rp) {
#pragma unroll
                for (int r = 0; r < 4; ++r) dst[r] = gv[r];
            }
        }
    }
}

// C = A B^T with the epilogue writing dtype T (dH) or accumulating fp32 (dW)
template <typename T, bool ACCUM>
__global__ void __launch_bounds__(THREADS) ce_gemm_kernel(const T *A, int64_t lda, int M, const T *B, int64_t ldb,
                                                         int N, int K, void *C, int64_t ldc) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    T *smem = reinterpret_cast<T *>(smem_raw);
    const int m0 = blockIdx.y * BM, n0 = blockIdx.x * BN;
    floatx4 acc[4][4];
    gemm_tile<T>(A + (int64_t)m0 * lda, lda, min(BM, M - m0), B + (int64_t)n0 * ldb, ldb, min(BN, N - n0), K, acc,
                 smem);
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
#pragma unroll
    for (int mi = 0; mi < 4; ++mi)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = m0 + 64 * wm + 16 * mi + 4 * g + r, n = n0 + 64 * wn + 16 * ni + l16;
                if (m < M && n < N) {
                    if (ACCUM) {
                        float *c = (float *)C + (int64_t)m * ldc + n;
                        *c += acc[mi][ni][r];
                    } else {
                        ((T *)C)[(int64_t)m * ldc + n] = from_f32<T>(acc[mi][ni][r]);
                    }
                }
            }
}

// Token scores in fp32, 256 x 128 tiles (or 128 x 64) on the bf16 matrix units: every value is split into
// three bf16 parts, x = hi + mid + lo with |mid| <= 2^-9 |x|, |lo| <= 2^-18 |x| and nothing
// left above 2^-27 |x|, and a product is the six part products down to 2^-18; the three
// left out are below 2^-26 of it, less than one fp32 rounding.  A k-step of 32 takes a
// wave (64 x 64) 96 MFMAs of 16 cycles, against 128 of 32 cycles with
// v_mfma_f32_16x16x4_f32.  Values are split on their way from registers to LDS, once a
// block, in the shadow of the MFMAs: 8 waves, two LDS buffers of three planes (72 KiB
// each) of 16-byte chunks, swizzled like the bf16 tiles; the loads run two steps ahead.
// 1000 x 8191 x 768 (12.6 GFLOP, one tile a CU): scores 65 us, G^T 68, dH 73, dW 81 (192
// blocks); with W, H and G^T transposed in memory for dH and dW 27 us more in all;
// the MFMAs run 48 % of the time, the rest is the first loads, the step's barrier and the
// epilogue.  The fp32 MFMAs took 172 us, parts made in front of the products 80.
// Rows past the end of an operand re-read its last row.  Infinite operands give NaN.
namespace split {
// S: a wave's 16 x 16 tiles along both axes; 4, or 2 for 128 x 64 tiles
template <int S> constexpr int tm() { return 64 * S; }
template <int S> constexpr int tn() { return 32 * S; }
constexpr int TM = tm<4>(), TN = tn<4>(), TT = 512;
// bf16 elements of a plane: A's tile, then B's (AT, BT: as they stand in memory, [K][M], [K][N],
// rows 16 elements apart from the next)
template <int S, bool AT> constexpr int a_tile() { return AT ? BK * (tm<S>() + 16) : tm<S>() * BK; }
template <int S, bool AT, bool BT> constexpr int plane() { return a_tile<S, AT>() + BK * (tn<S>() + (BT ? 16 : 0)); }
using U16 = unsigned short;

template <int S> struct Raw {
    uint4 a[S], b[S / 2];  // a thread's loads of a step
};

__device__ __forceinline__ int swz(int row, int c) { return c ^ ((row >> 1) & 3); }
// place of a row of a [32][..] tile: bits 2 and 3 swapped, so that the 32-byte pieces that
// half a wave reads (rows 0 .. 3 and 8 .. 11, or four or sixteen behind them) share no bank
__device__ __forceinline__ int place(int row) { return (row & 19) | (row & 4) << 1 | (row & 8) >> 1; }

template <int PLANE> __device__ __forceinline__ void store(uint4 raw, U16 *lds) {
    float v[4] = {__uint_as_float(raw.x), __uint_as_float(raw.y), __uint_as_float(raw.z), __uint_as_float(raw.w)};
#pragma unroll
    for (int part = 0; part < 3; ++part) {
        const uint2 q = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        *reinterpret_cast<uint2 *>(lds + part * PLANE) = q;
        v[0] -= __uint_as_float(q.x << 16);
        v[1] -= __uint_as_float(q.x & 0xFFFF0000u);
        v[2] -= __uint_as_float(q.y << 16);
        v[3] -= __uint_as_float(q.y & 0xFFFF0000u);
    }
}

// acc[mi][ni] lane holds C[16*S*(w>>1) + 16mi + 4g + r][16*S*(w&1) + 16ni + l16]; K % 32 == 0.
// Row strides below 2^22 (32-bit byte offsets in a tile).
// BT: B is [K][N] as it stands in memory, b_rows of its K rows there (past them A is zero)
// and b_cols columns (a multiple of four).  Its tile stays [32][N] in LDS, and the
// fragments come out by transpose reads.  AT: A alike, with every row and column of a tile
// in memory.
template <int S, bool AT, bool BT>
__device__ __forceinline__ void tile(const float *A, int64_t lda, int a_rows, const float *B, int64_t ldb, int b_rows, int b_cols,
                                     int K, floatx4 (&acc)[S][S], U16 *s0, U16 *s1) {
    constexpr int PLANE = plane<S, AT, BT>(), A_TILE = a_tile<S, AT>(), PA = tm<S>() + 16, PB = tn<S>() + 16;
    constexpr int PIECES = S + S / 2;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int arow0 = 16 * S * (w >> 1), bcol0 = 16 * S * (w & 1);
#pragma unroll
    for (int mi = 0; mi < S; ++mi)
#pragma unroll
        for (int ni = 0; ni < S; ++ni) acc[mi][ni] = floatx4{0.f, 0.f, 0.f, 0.f};
    // thread -> rows tid / 8 + 64 i, values 4 (tid % 8) ..: half a chunk of eight
    const int r8 = tid >> 3, c8 = tid & 7;
    unsigned ao[S], bo[S / 2];
#pragma unroll
    for (int i = 0; i < S; ++i) ao[i] = 4u * ((unsigned)min(r8 + 64 * i, a_rows - 1) * (unsigned)lda + 4 * c8);
#pragma unroll
    for (int i = 0; i < S / 2; ++i) bo[i] = 4u * ((unsigned)min(r8 + 64 * i, b_rows - 1) * (unsigned)ldb + 4 * c8);
    const int to = r8 * BK + 8 * swz(r8, c8 >> 1) + 4 * (c8 & 1);  // the swizzle repeats every eight rows
    // AT, BT: thread -> the tile's row tid / 16, columns 4 (tid % 16) + 64 i
    const int r16 = tid >> 4, c16 = tid & 15, at_to = place(r16) * PA + 4 * c16, bt_to = A_TILE + place(r16) * PB + 4 * c16;
    const unsigned at = 4u * ((unsigned)r16 * (unsigned)lda + 4 * c16);
#pragma unroll
    for (int i = 0; i < S / 2; ++i)
        if (BT) bo[i] = 4u * min(64 * i + 4 * c16, b_cols - 4);
    auto gload = [&](Raw<S> &x, int step) {
        const char *a = reinterpret_cast<const char *>(AT ? A + (int64_t)step * BK * lda : A + (int64_t)step * BK);
        const int row0 = BT ? min(step * BK, b_rows - 1) : 0;
        const char *b = reinterpret_cast<const char *>(BT ? B + row0 * ldb : B + (int64_t)step * BK);
        const unsigned row = BT ? 4u * (unsigned)min(r16, b_rows - 1 - row0) * (unsigned)ldb : 0u;
#pragma unroll
        for (int i = 0; i < S; ++i) x.a[i] = *reinterpret_cast<const uint4 *>(AT ? a + at + 256 * i : a + ao[i]);
#pragma unroll
        for (int i = 0; i < S / 2; ++i) x.b[i] = *reinterpret_cast<const uint4 *>(b + (row + bo[i]));
    };
    auto put = [&](const Raw<S> &x, U16 *s, int i) {
        const uint4 v = i < S ? x.a[i < S ? i : 0] : x.b[i < S ? 0 : i - S];
        if (i < S) store<PLANE>(v, s + (AT ? at_to + 64 * i : to + 64 * i * BK));
        else store<PLANE>(v, s + (BT ? bt_to + 64 * (i - S) : A_TILE + to + 64 * (i - S) * BK));
    };
    // AT, BT: the lane's column l16 of a 16-column chunk, k = 8 g ..: rows 8 g + l16 / 4 and four behind it
    const int row_t = place(8 * g + (l16 >> 2)), col_t = 4 * (l16 & 3);
    const int at_from = row_t * PA + arow0 + col_t, bt_from = A_TILE + row_t * PB + bcol0 + col_t;
    auto fragment_t = [&](const U16 *at, int pitch) {
        const shortx4 lo = lds_read_tr(at), hi = lds_read_tr(at + 8 * pitch);
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto fragment = [&](const U16 *s, int row, int part) {
        return *reinterpret_cast<const bf16x8 *>(s + part * PLANE + (row + l16) * BK + 8 * swz(l16, g));
    };
    // the products of the step in `cur`; the next step's values go from x to `next`
    auto step = [&](const U16 *cur, U16 *next, const Raw<S> &x) {
        bf16x8 a[S][3];
#pragma unroll
        for (int mi = 0; mi < S; ++mi)
#pragma unroll
            for (int part = 0; part < 3; ++part)
                a[mi][part] = AT ? fragment_t(cur + part * PLANE + at_from + 16 * mi, PA) : fragment(cur, arow0 + 16 * mi, part);
#pragma unroll
        for (int ni = 0; ni < S; ++ni) {
            bf16x8 b[3];
#pragma unroll
            for (int part = 0; part < 3; ++part)
                b[part] = BT ? fragment_t(cur + part * PLANE + bt_from + 16 * ni, PB) : fragment(cur + A_TILE, bcol0 + 16 * ni, part);
            constexpr int QA[6] = {2, 0, 1, 1, 0, 0}, QB[6] = {0, 2, 1, 0, 1, 0};  // small products first
#pragma unroll
            for (int j = 0; j < 6; ++j)
#pragma unroll
                for (int mi = 0; mi < S; ++mi)
                    acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[mi][QA[j]], b[QB[j]], acc[mi][ni], 0, 0, 0);
            if (ni < S - 1)
#pragma unroll
                for (int i = ni * PIECES / (S - 1); i < (ni + 1) * PIECES / (S - 1); ++i) put(x, next, i);
        }
    };
    const int KT = K / BK;
    Raw<S> x0, x1;
    gload(x0, 0);
    gload(x1, min(1, KT - 1));
#pragma unroll
    for (int i = 0; i < PIECES; ++i) put(x0, s0, i);
    __syncthreads();
    for (int kt = 0; kt < KT; kt += 2) {
        gload(x0, min(kt + 2, KT - 1));
        step(s0, s1, x1);
        __syncthreads();
        if (kt + 1 >= KT) break;
        gload(x1, min(kt + 3, KT - 1));
        step(s1, s0, x0);
        __syncthreads();
    }
}

template <int S>
__global__ void __launch_bounds__(TT) scores_tile_kernel(FwdParams p) {
    constexpr int TM = tm<S>(), TN = tn<S>();
    __shared__ __align__(16) U16 s0[3 * plane<S, false, false>()], s1[3 * plane<S, false, false>()];
    __shared__ float sM[2][TM], sS[2][TM], sT[2][TM];
    __shared__ __align__(16) int sToken[TM];
    const qpam_ce_fwd_args &a = p.a;
    const int vt = blockIdx.x, r0 = blockIdx.y * TM, v0 = vt * TN;
    if (threadIdx.x < TM) sToken[threadIdx.x] = row_token(p, r0 + threadIdx.x);
    floatx4 acc[S][S];
    tile<S, false, false>((const float *)a.h + (int64_t)r0 * a.ldh, a.ldh, min(TM, a.N - r0),
                          (const float *)a.w + (int64_t)v0 * a.ldw, a.ldw, min(TN, a.V - v0), 0, a.D, acc, s0, s1);
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1, vl = v0 + 16 * S * wn + l16;
#pragma unroll
    for (int mi = 0; mi < S; ++mi) {
        const intx4 token = *reinterpret_cast<const intx4 *>(&sToken[16 * S * wm + 16 * mi + 4 * g]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            keep_token(p, acc[mi], r, r0 + 16 * S * wm + 16 * mi + 4 * g + r, token[r], vl);
            float mx = -INFINITY;
#pragma unroll
            for (int ni = 0; ni < S; ++ni)
                if (vl + 16 * ni < a.V) mx = fmaxf(mx, acc[mi][ni][r]);
            const float m = row16_max(mx);
            float s = 0.f, t = 0.f;
#pragma unroll
            for (int ni = 0; ni < S; ++ni)
                if (vl + 16 * ni < a.V) {
                    const float d = acc[mi][ni][r] - m, e = __builtin_amdgcn_exp2f(d * p.c);
                    s += e;
                    t = __builtin_fmaf(e, d, t);
                }
            s = row16_sum(s);
            t = row16_sum(t);
            if (l16 == 0) {
                const int row = 16 * S * wm + 16 * mi + 4 * g + r;
                sM[wn][row] = m;
                sS[wn][row] = s;
                sT[wn][row] = t * p.c;
            }
        }
    }
    __syncthreads();
    if (tid < TM && r0 + tid < a.N) {
        float m = sM[0][tid], s = sS[0][tid], t = sT[0][tid];
        join_scores(p.c, m, s, t, sM[1][tid], sS[1][tid], sT[1][tid]);
        const int64_t o = (int64_t)(r0 + tid) * p.n_vt + vt;
        p.part_m[o] = m;
        p.part_s[o] = s;
        p.part_t[o] = t;
    }
}

// G^T [Vp][Rp] without the tokens' one-hot terms; zero past the vocabulary and past the rows
// (Rp: a multiple of 256)
template <int S>
__global__ void __launch_bounds__(TT) scores_grad_kernel(BwdParams p) {
    constexpr int TM = tm<S>(), TN = tn<S>();
    __shared__ __align__(16) U16 s0[3 * plane<S, false, false>()], s1[3 * plane<S, false, false>()];
    __shared__ __align__(16) float sRow[3][TM];
    const qpam_ce_bwd_args &a = p.a;
    const int lr0 = blockIdx.y * TM, v0 = blockIdx.x * TN, tid = threadIdx.x;
    if (tid < TM) {
        const RowScore q = row_score(p, lr0 + tid);
        sRow[0][tid] = q.m;
        sRow[1][tid] = q.base;
        sRow[2][tid] = q.slope;
    }
    floatx4 acc[S][S];
    // a tile of padding alone (the small ones) reads the last row
    const int lr = min(lr0, p.rows - 1), vr = min(v0, a.V - 1);
    tile<S, false, false>((const float *)a.h + (int64_t)(p.row0 + lr) * a.ldh, a.ldh, min(TM, p.rows - lr),
                          (const float *)a.w + (int64_t)vr * a.ldw, a.ldw, min(TN, a.V - vr), 0, a.D, acc, s0, s1);
    const int w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
    float *GT = (float *)p.gtbuf;
#pragma unroll
    for (int mi = 0; mi < S; ++mi) {
        const int rl = 16 * S * wm + 16 * mi + 4 * g;
        const floatx4 hm = *reinterpret_cast<const floatx4 *>(&sRow[0][rl]);
        const floatx4 h0 = *reinterpret_cast<const floatx4 *>(&sRow[1][rl]);
        const floatx4 h1 = *reinterpret_cast<const floatx4 *>(&sRow[2][rl]);
#pragma unroll
        for (int ni = 0; ni < S; ++ni) {
            const int v = v0 + 16 * S * wn + 16 * ni + l16;
            floatx4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float u = score_u(acc[mi][ni][r], hm[r], p.c);
                const bool in = v < a.V && lr0 + rl + r < p.rows;
                x[r] = in ? __builtin_amdgcn_exp2f(u) * __builtin_fmaf(h1[r], u, h0[r]) : 0.f;
            }
            *reinterpret_cast<floatx4 *>(GT + (int64_t)v * p.Rp + lr0 + rl) = x;
        }
    }
}

// C = A B, B [b_rows][N] with b_rows <= K and zeros in A past them, A [M][K] (dW: G^T) or
// with AT [K][M] (dH: G^T again).  The K axis in gridDim.z ranges of kper: one range writes
// C (or adds to it), several write C + z split_stride, summed by sum_kernel in their order.
template <bool AT>
__global__ void __launch_bounds__(TT) gemm_kernel(const float *A, int64_t lda, int M, const float *B, int64_t ldb, int b_rows,
                                                  int N, int K, int kper, float *C, int64_t ldc, int64_t split_stride, int accumulate) {
    __shared__ __align__(16) U16 s0[3 * plane<4, AT, true>()], s1[3 * plane<4, AT, true>()];
    const int m0 = blockIdx.y * TM, n0 = blockIdx.x * TN, k0 = blockIdx.z * kper;
    floatx4 acc[4][4];
    const int kb = min(k0, b_rows - 1);  // a range past B's rows: A is zero there
    tile<4, AT, true>(AT ? A + (int64_t)k0 * lda + m0 : A + (int64_t)m0 * lda + k0, lda, min(TM, M - m0), B + (int64_t)kb * ldb + n0, ldb, b_rows - kb, min(TN, N - n0),
               min(kper, K - k0), acc, s0, s1);
    C += blockIdx.z * split_stride;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
#pragma unroll
    for (int mi = 0; mi < 4; ++mi)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = m0 + 64 * wm + 16 * mi + 4 * g + r, n = n0 + 64 * wn + 16 * ni + l16;
                if (m < M && n < N) {
                    float *c = C + (int64_t)m * ldc + n;
                    *c = accumulate ? *c + acc[mi][ni][r] : acc[mi][ni][r];
                }
            }
}

// rows * cols is below 2^24 where there are several ranges; cols % 4 == 0
template <typename T>
__global__ void __launch_bounds__(THREADS) sum_kernel(const float *part, int ranges, int rows, int cols, T *out, int64_t ldo,
                                                      int accumulate) {
    const unsigned n4 = (unsigned)rows * (unsigned)cols / 4, per_row = cols / 4;
    for (unsigned i = blockIdx.x * THREADS + threadIdx.x; i < n4; i += gridDim.x * THREADS) {
        floatx4 x = reinterpret_cast<const floatx4 *>(part)[i];
#pragma unroll 4
        for (int z = 1; z < ranges; ++z) x += reinterpret_cast<const floatx4 *>(part)[(int64_t)z * n4 + i];
        const unsigned r = i / per_row;
        T *to = out + r * ldo + 4 * (i - r * per_row);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float y = accumulate ? Elem<T>::load(to + j) + x[j] : x[j];
            if constexpr (sizeof(T) == 2) to[j] = __builtin_bit_cast(unsigned short, (__bf16)y);
            else to[j] = y;
        }
    }
}

// 128 x 64 tiles (two blocks a CU) up to 128 tiles of 256 x 128, which leave half the CUs
// idle.  Scores at D = 768, small against large: 12 tiles 24 and 52 us, 64 tiles 28 and 53,
// 126 tiles 45 and 57, 160 tiles 61 and 58, 256 tiles 82 and 66.
inline bool small_tiles(int64_t M, int64_t N) { return ((M + TM - 1) / TM) * ((N + TN - 1) / TN) <= 128; }
}  // namespace split

// ------------------------------------------------------ bf16 big tiles ----
// bf16 operands use 256 x 256 block tiles: 4 waves of 128 x 128, 8 x 8
// accumulator tiles (256 fp32 per lane, AGPR resident), 64 MFMA per 32-wide
// k-step against 16 fragment reads (64 flops per LDS byte), global loads
// prefetched two k-steps ahead through registers into a double-buffered LDS.
namespace big {
constexpr int BTM = 256;                // block tile rows (A operand)
constexpr int BTN = 128;                // block tile cols (B operand)
constexpr int PITCH = BK + 8;           // bf16 elements per LDS row
constexpr int LOADS_A = BTM * 4 / THREADS;  // 16-byte loads per thread per k-step
constexpr int LOADS_B = BTN * 4 / THREADS;
constexpr size_t SMEM = (size_t)2 * (BTM + BTN) * PITCH * sizeof(unsigned short);  // 60 KiB
using U16 = unsigned short;

struct Frag {
    uint4 a[LOADS_A], b[LOADS_B];
};

// Workgroups are dispatched round-robin over the 8 XCDs, each with its own L2.
// Give every XCD a contiguous range of work items (grid = 8 * per; items >=
// total are idle) so that concurrently running tiles of one XCD share rows.
constexpr int XCDS = 8;
__device__ __forceinline__ int xcd_item(int bid, int total) {
    const int per = (total + XCDS - 1) / XCDS;
    return (bid % XCDS) * per + bid / XCDS;
}
inline int xcd_grid(int total) { return XCDS * ((total + XCDS - 1) / XCDS); }

// Item -> (row tile, col tile), grouping GM row tiles: consecutive items walk
// the GM row tiles of one column tile, then the next column tile, so a window
// of ~32 items touches GM row tiles and ~32/GM column tiles.
constexpr int GM = 4;
__device__ __forceinline__ void grouped_tile(int item, int n_rt, int n_ct, int &rt, int &ct) {
    const int group = item / (GM * n_ct);
    const int in_group = item - group * GM * n_ct;
    const int rows = min(GM, n_rt - group * GM);
    rt = group * GM + in_group % rows;
    ct = in_group / rows;
}

__device__ __forceinline__ void gload(Frag &f, const U16 *A, int64_t lda, int a_rows, const U16 *B, int64_t ldb,
                                      int b_rows, int k0) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < LOADS_A; ++i) {
        const int ci = tid + i * THREADS, row = ci >> 2, c = ci & 3;
        f.a[i] = (row < a_rows) ? *reinterpret_cast<const uint4 *>(A + row * lda + k0 + 8 * c) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < LOADS_B; ++i) {
        const int ci = tid + i * THREADS, row = ci >> 2, c = ci & 3;
        f.b[i] = (row < b_rows) ? *reinterpret_cast<const uint4 *>(B + row * ldb + k0 + 8 * c) : make_uint4(0, 0, 0, 0);
    }
}

__device__ __forceinline__ void lstore(const Frag &f, U16 *sA, U16 *sB) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < LOADS_A; ++i) {
        const int ci = tid + i * THREADS, row = ci >> 2, c = ci & 3;
        *reinterpret_cast<uint4 *>(sA + row * PITCH + 8 * c) = f.a[i];
    }
#pragma unroll
    for (int i = 0; i < LOADS_B; ++i) {
        const int ci = tid + i * THREADS, row = ci >> 2, c = ci & 3;
        *reinterpret_cast<uint4 *>(sB + row * PITCH + 8 * c) = f.b[i];
    }
}

__device__ __forceinline__ void mma_step(const U16 *sA, const U16 *sB, floatx4 (&acc)[8][4], int arow0, int brow0,
                                         int l16, int g) {
    // B fragments stay in registers for the step; A fragments are read per row tile
    bf16x8 bfr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) bfr[i] = *reinterpret_cast<const bf16x8 *>(sB + (brow0 + 16 * i + l16) * PITCH + 8 * g);
#pragma unroll
    for (int mi = 0; mi < 8; ++mi) {
        const bf16x8 af = *reinterpret_cast<const bf16x8 *>(sA + (arow0 + 16 * mi + l16) * PITCH + 8 * g);
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
            acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, bfr[ni], acc[mi][ni], 0, 0, 0);
    }
}

// C[m][n] = sum_{k in [k_begin, k_end)} A[m][k] B[n][k] for one 256 x 128 tile.
// acc[mi][ni] lane holds C[128*(w>>1) + 16mi + 4g + r][64*(w&1) + 16ni + l16].
// DEEP prefetches two k-steps ahead (two register stages); otherwise one.
template <bool DEEP>
__device__ __forceinline__ void gemm_tile(const U16 *A, int64_t lda, int a_rows, const U16 *B, int64_t ldb,
                                          int b_rows, int k_begin, int k_end, floatx4 (&acc)[8][4], U16 *smem) {
    U16 *sA[2] = {smem, smem + (BTM + BTN) * PITCH};
    U16 *sB[2] = {smem + BTM * PITCH, smem + (BTM + BTN) * PITCH + BTM * PITCH};
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int arow0 = 128 * (w >> 1), brow0 = 64 * (w & 1);
#pragma unroll
    for (int mi = 0; mi < 8; ++mi)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int KT = (k_end - k_begin) / BK;
    if (KT <= 0) return;
    if (!DEEP) {
        Frag f;
        gload(f, A, lda, a_rows, B, ldb, b_rows, k_begin);
        lstore(f, sA[0], sB[0]);
        __syncthreads();
        for (int kt = 0; kt < KT; ++kt) {
            const int buf = kt & 1;
            if (kt + 1 < KT) gload(f, A, lda, a_rows, B, ldb, b_rows, k_begin + (kt + 1) * BK);
            mma_step(sA[buf], sB[buf], acc, arow0, brow0, l16, g);
            if (kt + 1 < KT) lstore(f, sA[buf ^ 1], sB[buf ^ 1]);
            __syncthreads();
        }
        return;
    }
    Frag f0, f1;
    gload(f0, A, lda, a_rows, B, ldb, b_rows, k_begin);
    if (KT > 1) gload(f1, A, lda, a_rows, B, ldb, b_rows, k_begin + BK);
    lstore(f0, sA[0], sB[0]);
    __syncthreads();
    for (int kt = 0; kt < KT; kt += 2) {
        // even step: tile kt in buffer 0, tile kt+1 waiting in f1
        if (kt + 2 < KT) gload(f0, A, lda, a_rows, B, ldb, b_rows, k_begin + (kt + 2) * BK);
        mma_step(sA[0], sB[0], acc, arow0, brow0, l16, g);
        if (kt + 1 < KT) lstore(f1, sA[1], sB[1]);
        __syncthreads();
        if (kt + 1 >= KT) break;
        // odd step: tile kt+1 in buffer 1, tile kt+2 waiting in f0
        if (kt + 3 < KT) gload(f1, A, lda, a_rows, B, ldb, b_rows, k_begin + (kt + 3) * BK);
        mma_step(sA[1], sB[1], acc, arow0, brow0, l16, g);
        if (kt + 2 < KT) lstore(f0, sA[0], sB[0]);
        __syncthreads();
    }
}

// forward: per (256 rows, 128 vocab) tile -> per-row (max, sum exp, argmax)
__global__ void __launch_bounds__(THREADS, 2) fwd_tile_kernel(FwdParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float sM[2][BTM], sS[2][BTM];
    __shared__ int sI[2][BTM];
    const qpam_ce_fwd_args &a = p.a;
    const int n_rt = (a.N + BTM - 1) / BTM;
    const int item = xcd_item(blockIdx.x, n_rt * p.n_vt);
    if (item >= n_rt * p.n_vt) return;
    int rt, vt;
    grouped_tile(item, n_rt, p.n_vt, rt, vt);
    const int r0 = rt * BTM, v0 = vt * BTN;
    floatx4 acc[8][4];
    gemm_tile<true>((const U16 *)a.h + (int64_t)r0 * a.ldh, a.ldh, min(BTM, a.N - r0), (const U16 *)a.w + (int64_t)v0 * a.ldw,
              a.ldw, min(BTN, a.V - v0), 0, a.D, acc, reinterpret_cast<U16 *>(smem_raw));
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
#pragma unroll
    for (int mi = 0; mi < 8; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float mx = -INFINITY;
            int ix = 0x7fffffff;
#pragma unroll
            for (int ni = 0; ni < 4; ++ni) {
                const int v = v0 + 64 * wn + 16 * ni + l16;
                const float x = (v < a.V) ? acc[mi][ni][r] : -INFINITY;
                if (x > mx) { mx = x; ix = v; }
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) {
                const float om = __shfl_xor(mx, off);
                const int oi = __shfl_xor(ix, off);
                if (om > mx || (om == mx && oi < ix)) { mx = om; ix = oi; }
            }
            float s = 0.f;
#pragma unroll
            for (int ni = 0; ni < 4; ++ni) {
                const int v = v0 + 64 * wn + 16 * ni + l16;
                if (v < a.V) s += __expf(acc[mi][ni][r] - mx);
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1) s += __shfl_xor(s, off);
            if (l16 == 0) {
                const int row = 128 * wm + 16 * mi + 4 * g + r;
                sM[wn][row] = mx;
                sS[wn][row] = s;
                sI[wn][row] = ix;
            }
        }
    }
    __syncthreads();
    if (r0 + tid < a.N) {
        const float m0 = sM[0][tid], m1 = sM[1][tid];
        const float m = fmaxf(m0, m1);
        float s = 0.f;
        if (m0 > -INFINITY) s += sS[0][tid] * __expf(m0 - m);
        if (m1 > -INFINITY) s += sS[1][tid] * __expf(m1 - m);
        const int i = (m1 > m0 || (m1 == m0 && sI[1][tid] < sI[0][tid])) ? sI[1][tid] : sI[0][tid];
        const int64_t o = (int64_t)(r0 + tid) * p.n_vt + vt;
        p.part_m[o] = m;
        p.part_s[o] = s;
        p.part_i[o] = i;
    }
}

// backward G tile (256 rows x 128 vocab): recompute logits, write G and G^T
__global__ void __launch_bounds__(THREADS, 2) grad_tile_kernel(BwdParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float sLse[BTM], sScale[BTM];
    __shared__ int sTgt[BTM];
    const qpam_ce_bwd_args &a = p.a;
    const int n_rt = p.Rp / BTM, n_vt = p.Vp / BTN;
    const int item = xcd_item(blockIdx.x, n_rt * n_vt);
    if (item >= n_rt * n_vt) return;
    int rt, vt;
    grouped_tile(item, n_rt, n_vt, rt, vt);
    const int lr0 = rt * BTM, v0 = vt * BTN;
    const int tid = threadIdx.x;
    {
        const int lr = lr0 + tid, row = p.row0 + lr;
        float lse = 0.f, sc = 0.f;
        int tg = -1;
        if (lr < p.rows) {
            const int64_t t = a.targets[row];
            const bool valid = (t != a.ignore_index) && t >= 0 && t < a.V;
            lse = a.lse[row];
            sc = valid ? a.grad_scale[0] * (a.mask ? a.mask[row] : 1.f) : 0.f;
            tg = valid ? (int)t : -1;
        }
        sLse[tid] = lse;
        sScale[tid] = sc;
        sTgt[tid] = tg;
    }
    floatx4 acc[8][4];
    gemm_tile<false>((const U16 *)a.h + (int64_t)(p.row0 + lr0) * a.ldh, a.ldh, min(BTM, p.rows - lr0),
              (const U16 *)a.w + (int64_t)v0 * a.ldw, a.ldw, min(BTN, a.V - v0), 0, a.D, acc,
              reinterpret_cast<U16 *>(smem_raw));
    const int w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
    U16 *G = (U16 *)p.gbuf;
    U16 *GT = (U16 *)p.gtbuf;
#pragma unroll
    for (int mi = 0; mi < 8; ++mi) {
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) {
            const int v = v0 + 64 * wn + 16 * ni + l16;
            const int rl0 = 128 * wm + 16 * mi + 4 * g;
            ushortx4 gv;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int rl = rl0 + r;
                float x = 0.f;
                if (v < a.V && sScale[rl] != 0.f) {
                    x = __expf(acc[mi][ni][r] - sLse[rl]);
                    if (v == sTgt[rl]) x -= 1.f;
                    x *= sScale[rl];
                }
                gv[r] = f32_to_bf16(x);
                if (p.write_g && lr0 + rl < p.rows) G[(int64_t)(lr0 + rl) * p.Vp + v] = gv[r];
            }
            *reinterpret_cast<ushortx4 *>(GT + (int64_t)v * p.Rp + lr0 + rl0) = gv;
        }
    }
}

// backward GEMMs: dW tiles (dW[v][d] += sum_r G^T[v][r] H^T[d][r]) and
// split-K partials of dH (dH_s[r][d] = sum_{v in split s} G[r][v] W^T[d][v])
// into fp32, as two kernels so each keeps two waves per SIMD.
struct GroupParams {
    BwdParams p;
    int n_dw, dw_ntiles_n;     // dW tiles, tiles along D
    int dh_ntiles_m, dh_ntiles_n, splits, ksplit;
    float *dh_part;            // [splits][rows][D]
};

__global__ void __launch_bounds__(THREADS, 2) dw_gemm_kernel(GroupParams q) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const BwdParams &p = q.p;
    const qpam_ce_bwd_args &a = p.a;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
    floatx4 acc[8][4];
    const int bid = xcd_item(blockIdx.x, q.n_dw);
    if (bid >= q.n_dw) return;
    const int mt = bid / q.dw_ntiles_n, nt = bid % q.dw_ntiles_n;
    const int m0 = mt * BTM, n0 = nt * BTN;
    gemm_tile<false>((const U16 *)p.gtbuf + (int64_t)m0 * p.Rp, p.Rp, min(BTM, a.V - m0),
              (const U16 *)p.ht + (int64_t)n0 * p.Rp, p.Rp, min(BTN, a.D - n0), 0, p.Rp, acc,
              reinterpret_cast<U16 *>(smem_raw));
#pragma unroll
    for (int mi = 0; mi < 8; ++mi)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = m0 + 128 * wm + 16 * mi + 4 * g + r, n = n0 + 64 * wn + 16 * ni + l16;
                if (m < a.V && n < a.D) static_cast<float *>(a.dw)[(int64_t)m * a.lddw + n] += acc[mi][ni][r];
            }
}

__global__ void __launch_bounds__(THREADS, 2) dh_gemm_kernel(GroupParams q) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    const BwdParams &p = q.p;
    const qpam_ce_bwd_args &a = p.a;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
    floatx4 acc[8][4];
    const int total = q.splits * q.dh_ntiles_m * q.dh_ntiles_n;
    const int bid = xcd_item(blockIdx.x, total);
    if (bid >= total) return;
    const int s = bid / (q.dh_ntiles_m * q.dh_ntiles_n);
    const int t = bid % (q.dh_ntiles_m * q.dh_ntiles_n);
    const int mt = t / q.dh_ntiles_n, nt = t % q.dh_ntiles_n;
    const int m0 = mt * BTM, n0 = nt * BTN;
    const int kb = s * q.ksplit, ke = min(p.Vp, kb + q.ksplit);
    gemm_tile<false>((const U16 *)p.gbuf + (int64_t)m0 * p.Vp, p.Vp, min(BTM, p.rows - m0),
              (const U16 *)p.wt + (int64_t)n0 * p.Vp, p.Vp, min(BTN, a.D - n0), kb, ke, acc,
              reinterpret_cast<U16 *>(smem_raw));
    float *dst = q.dh_part + (int64_t)s * p.rows * a.D;
#pragma unroll
    for (int mi = 0; mi < 8; ++mi)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int m = m0 + 128 * wm + 16 * mi + 4 * g + r, n = n0 + 64 * wn + 16 * ni + l16;
                if (m < p.rows && n < a.D) dst[(int64_t)m * a.D + n] = acc[mi][ni][r];
            }
}

// dH rows of the chunk = sum of the split partials, written as bf16
__global__ void __launch_bounds__(THREADS) dh_reduce_kernel(GroupParams q) {
    const BwdParams &p = q.p;
    const qpam_ce_bwd_args &a = p.a;
    const int64_t n = (int64_t)p.rows * a.D;
    for (int64_t e = blockIdx.x * (int64_t)THREADS + threadIdx.x; e < n; e += (int64_t)gridDim.x * THREADS) {
        float x = 0.f;
        for (int s = 0; s < q.splits; ++s) x += q.dh_part[s * n + e];
        const int64_t r = e / a.D, c = e - r * a.D;
        reinterpret_cast<U16 *>(a.dh)[(int64_t)(p.row0 + r) * a.lddh + c] = f32_to_bf16(x);
    }
}

constexpr int DH_SPLITS = 8;
}  // namespace big

// 256 x 256 tiles for the bf16 logits GEMMs (hidden size a multiple of 64): one
// block of 4 waves per tile, each wave a 128 x 128 quadrant (64 accumulator
// tiles, one wave per SIMD), k-steps of 64 through double-buffered LDS (72 KiB
// per stage) with the next stage's global loads in flight in registers.  Rows
// past the end of an operand re-read its last row (the epilogues mask them), so
// the pipelined loads carry no conditional register initialisation.
namespace wide {
constexpr int TM = 256, TN = 256, WK = 64;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int WTHREADS = 512;   // 8 waves: 4 row groups x 2 column groups, 64 x 128 each
constexpr int WPITCH = WK + 8;  // bf16 elements per LDS row (144 bytes: conflict-free 16-byte reads)
constexpr int WLOADS = TM * WK / 8 / WTHREADS;  // 16-byte loads per thread per operand per k-step (4)
constexpr size_t WSMEM = (size_t)2 * (TM + TN) * WPITCH * sizeof(unsigned short);  // 144 KiB
using U16 = unsigned short;

struct WFrag {
    uintx4 a[WLOADS], b[WLOADS];
};

// Rows past the end of an operand re-read its last row (the epilogues mask them).
// Addresses are a wave-uniform base plus a 32-bit byte offset per load.
__device__ __forceinline__ void wgload(WFrag &f, const U16 *A, int64_t lda, int a_rows, const U16 *B, int64_t ldb,
                                       int b_rows, int k0) {
    const int tid = threadIdx.x, c8 = 8 * (tid & 7);
    const char *ab = reinterpret_cast<const char *>(A + k0), *bb = reinterpret_cast<const char *>(B + k0);
#pragma unroll
    for (int i = 0; i < WLOADS; ++i) {
        const int row = (tid >> 3) + 64 * i;
        const unsigned ao = 2u * (unsigned)(min(row, a_rows - 1) * (int)lda + c8);
        const unsigned bo = 2u * (unsigned)(min(row, b_rows - 1) * (int)ldb + c8);
        f.a[i] = *reinterpret_cast<const uintx4 *>(ab + ao);
        f.b[i] = *reinterpret_cast<const uintx4 *>(bb + bo);
    }
}

__device__ __forceinline__ void wlstore(const WFrag &f, U16 *sA, U16 *sB) {
    const int tid = threadIdx.x, c8 = 8 * (tid & 7);
#pragma unroll
    for (int i = 0; i < WLOADS; ++i) {
        const int row = (tid >> 3) + 64 * i;
        *reinterpret_cast<uintx4 *>(sA + row * WPITCH + c8) = f.a[i];
        *reinterpret_cast<uintx4 *>(sB + row * WPITCH + c8) = f.b[i];
    }
}

// One k-step (64) of the wave's 64 x 128 block: per 32-wide half, the four A
// fragments stay in registers while the eight B fragments stream through (each
// feeds four MFMAs).
__device__ __forceinline__ void wmma_stage(const U16 *sA, const U16 *sB, floatx4 (&acc)[4][8], int arow0, int brow0,
                                           int l16, int g) {
#pragma unroll
    for (int ks = 0; ks < WK / 32; ++ks) {
        bf16x8 af[4];
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
            af[mi] = *reinterpret_cast<const bf16x8 *>(sA + (arow0 + 16 * mi + l16) * WPITCH + 32 * ks + 8 * g);
#pragma unroll
        for (int ni = 0; ni < 8; ++ni) {
            const bf16x8 bfr = *reinterpret_cast<const bf16x8 *>(sB + (brow0 + 16 * ni + l16) * WPITCH + 32 * ks + 8 * g);
#pragma unroll
            for (int mi = 0; mi < 4; ++mi)
                acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[mi], bfr, acc[mi][ni], 0, 0, 0);
        }
    }
}

// C[m][n] = sum_k A[m][k] B[n][k] (k in [0, K), K a multiple of 64) for one 256 x 256
// tile; acc[mi][ni] lane holds C[64*(w>>1) + 16mi + 4g + r][128*(w&1) + 16ni + l16].
// The global loads of k-step kt + 1 are issued (and pinned) before the MFMAs of
// k-step kt and reach the other LDS buffer after them; the second wave on each
// SIMD covers the rest of their latency.
__device__ __forceinline__ void wgemm_tile(const U16 *A, int64_t lda, int a_rows, const U16 *B, int64_t ldb,
                                           int b_rows, int K, floatx4 (&acc)[4][8], U16 *smem) {
    U16 *sA0 = smem, *sB0 = smem + TM * WPITCH;
    U16 *sA1 = smem + (TM + TN) * WPITCH, *sB1 = sA1 + TM * WPITCH;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int arow0 = 64 * (w >> 1), brow0 = 128 * (w & 1);
#pragma unroll
    for (int mi = 0; mi < 4; ++mi)
#pragma unroll
        for (int ni = 0; ni < 8; ++ni) acc[mi][ni] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int KT = K / WK;
    WFrag f;
    wgload(f, A, lda, a_rows, B, ldb, b_rows, 0);
    wlstore(f, sA0, sB0);
    __syncthreads();
    // two k-steps per iteration (buffers by compile-time index); the loads are
    // unconditional (past the end they re-read the last k-step) so that every path
    // has the same memory operations
    int kt = 0;
    for (; kt + 1 < KT; kt += 2) {
        wgload(f, A, lda, a_rows, B, ldb, b_rows, (kt + 1) * WK);
        __builtin_amdgcn_sched_barrier(0);
        wmma_stage(sA0, sB0, acc, arow0, brow0, l16, g);
        __builtin_amdgcn_sched_barrier(0);
        wlstore(f, sA1, sB1);
        __syncthreads();
        wgload(f, A, lda, a_rows, B, ldb, b_rows, min(kt + 2, KT - 1) * WK);
        __builtin_amdgcn_sched_barrier(0);
        wmma_stage(sA1, sB1, acc, arow0, brow0, l16, g);
        __builtin_amdgcn_sched_barrier(0);
        wlstore(f, sA0, sB0);
        __syncthreads();
    }
    if (kt < KT) wmma_stage(sA0, sB0, acc, arow0, brow0, l16, g);
}

// The same tile product with the operands streamed global -> LDS by direct
// (no register) loads: four LDS stages of k = 32 (128 KiB), the loads of k-step
// kt + 3 issued when k-step kt starts, so each load has three k-steps to land.
// Each direct load writes 64 lanes x 16 bytes = 16 rows x 64 bytes contiguously;
// the 16-byte chunks of a row are XOR-swizzled (chunk c of row r at c ^ ((r >> 1) & 3))
// so that the fragment reads (16 rows, one chunk) hit distinct banks.  Separate
// arrays per stage let the compiler's memory-counter tracking tell the stages apart;
// the wait before each barrier is explicit: every k-step issues exactly four
// direct loads per wave (past the end they re-read the last k-step into a free
// stage), so "own loads of the next k-step done" is vmcnt <= 8.
constexpr int DK = 32, DSTAGES = 4;
constexpr bool USE_DMA = true;                  // direct-load mainloop (else register-staged)
constexpr size_t KSMEM = USE_DMA ? 0 : WSMEM;   // dynamic LDS of the tile kernels
__device__ __forceinline__ int swz(int row, int c) { return c ^ ((row >> 1) & 3); }

template <int S>
__device__ __forceinline__ void dma_stage(U16 (&sA)[TM * DK], U16 (&sB)[TN * DK], const U16 *A, int64_t lda,
                                          int a_rows, const U16 *B, int64_t ldb, int b_rows, int k0) {
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r0 = 32 * w + 16 * j, row = r0 + (lane >> 2), c = swz(row, lane & 3);
        __builtin_amdgcn_global_load_lds(A + (int64_t)min(row, a_rows - 1) * lda + k0 + 8 * c, &sA[r0 * DK], 16, 0, 0);
        __builtin_amdgcn_global_load_lds(B + (int64_t)min(row, b_rows - 1) * ldb + k0 + 8 * c, &sB[r0 * DK], 16, 0, 0);
    }
}

__device__ __forceinline__ void dma_mma(const U16 *sA, const U16 *sB, floatx4 (&acc)[4][8], int arow0, int brow0,
                                        int l16, int g) {
    bf16x8 af[4];
#pragma unroll
    for (int mi = 0; mi < 4; ++mi) {
        const int row = arow0 + 16 * mi + l16;
        af[mi] = *reinterpret_cast<const bf16x8 *>(sA + row * DK + 8 * swz(row, g));
    }
#pragma unroll
    for (int ni = 0; ni < 8; ++ni) {
        const int row = brow0 + 16 * ni + l16;
        const bf16x8 bfr = *reinterpret_cast<const bf16x8 *>(sB + row * DK + 8 * swz(row, g));
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
            acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[mi], bfr, acc[mi][ni], 0, 0, 0);
    }
}

__device__ __forceinline__ void wgemm_tile_dma(const U16 *A, int64_t lda, int a_rows, const U16 *B, int64_t ldb,
                                               int b_rows, int K, floatx4 (&acc)[4][8]) {
    __shared__ __align__(16) U16 sA0[TM * DK], sA1[TM * DK], sA2[TM * DK], sA3[TM * DK];
    __shared__ __align__(16) U16 sB0[TN * DK], sB1[TN * DK], sB2[TN * DK], sB3[TN * DK];
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int arow0 = 64 * (w >> 1), brow0 = 128 * (w & 1);
#pragma unroll
    for (int mi = 0; mi < 4; ++mi)
#pragma unroll
        for (int ni = 0; ni < 8; ++ni) acc[mi][ni] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int KT = K / DK;
    dma_stage<0>(sA0, sB0, A, lda, a_rows, B, ldb, b_rows, 0);
    dma_stage<1>(sA1, sB1, A, lda, a_rows, B, ldb, b_rows, min(1, KT - 1) * DK);
    dma_stage<2>(sA2, sB2, A, lda, a_rows, B, ldb, b_rows, min(2, KT - 1) * DK);
    stage_barrier<8>();
#define QPAM_DMA_STEP(KT_, CUR_A, CUR_B, NXT_A, NXT_B, NS)                                                    \
    dma_stage<NS>(NXT_A, NXT_B, A, lda, a_rows, B, ldb, b_rows, min((KT_) + 3, KT - 1) * DK);                 \
    __builtin_amdgcn_sched_barrier(0);                                                                         \
    dma_mma(CUR_A, CUR_B, acc, arow0, brow0, l16, g);                                                          \
    stage_barrier<8>();
    int kt = 0;
    for (; kt + 3 < KT; kt += 4) {
        QPAM_DMA_STEP(kt, sA0, sB0, sA3, sB3, 3)
        QPAM_DMA_STEP(kt + 1, sA1, sB1, sA0, sB0, 0)
        QPAM_DMA_STEP(kt + 2, sA2, sB2, sA1, sB1, 1)
        QPAM_DMA_STEP(kt + 3, sA3, sB3, sA2, sB2, 2)
    }
    if (kt < KT) { QPAM_DMA_STEP(kt, sA0, sB0, sA3, sB3, 3) }
    if (kt + 1 < KT) { QPAM_DMA_STEP(kt + 1, sA1, sB1, sA0, sB0, 0) }
    if (kt + 2 < KT) { QPAM_DMA_STEP(kt + 2, sA2, sB2, sA1, sB1, 1) }
#undef QPAM_DMA_STEP
    // drain the direct loads still in flight before the LDS is reused or the wave ends
    __builtin_amdgcn_s_waitcnt(0 | 0x70 | 0xF00);
}

__device__ __forceinline__ int xcd_item(int bid, int total) { return big::xcd_item(bid, total); }

// Order a wave's LDS accesses around a point: its earlier LDS operations are
// complete (lgkmcnt 0) and no LDS access moves across it.
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0), vmcnt / expcnt unconstrained
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// forward: per (256 rows, 256 vocab) tile -> per-row (max, sum exp[, argmax]).
// Row statistics over a wave's 128 columns: per lane over its 8 columns, then
// across the 16 lanes that hold the row (DPP); the argmax (first column at the
// maximum) only when accuracy counts are requested.
template <bool ARGMAX>
__global__ void __launch_bounds__(WTHREADS) fwd_tile_kernel(FwdParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float sM[2][TM], sS[2][TM];
    __shared__ int sI[2][TM];
    const qpam_ce_fwd_args &a = p.a;
    const int n_rt = (a.N + TM - 1) / TM;
    const int item = xcd_item(blockIdx.x, n_rt * p.n_vt);
    if (item >= n_rt * p.n_vt) return;
    int rt, vt;
    big::grouped_tile(item, n_rt, p.n_vt, rt, vt);
    const int r0 = rt * TM, v0 = vt * TN;
    floatx4 acc[4][8];
    if constexpr (USE_DMA)
        wgemm_tile_dma((const U16 *)a.h + (int64_t)r0 * a.ldh, a.ldh, min(TM, a.N - r0),
                       (const U16 *)a.w + (int64_t)v0 * a.ldw, a.ldw, min(TN, a.V - v0), a.D, acc);
    else
        wgemm_tile((const U16 *)a.h + (int64_t)r0 * a.ldh, a.ldh, min(TM, a.N - r0),
                   (const U16 *)a.w + (int64_t)v0 * a.ldw, a.ldw, min(TN, a.V - v0), a.D, acc,
                   reinterpret_cast<U16 *>(smem_raw));
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
    const int vl = v0 + 128 * wn + l16;  // this lane's column in tile ni: vl + 16 ni
    const bool full = v0 + TN <= a.V;    // no column past the vocabulary: no per-element checks
#pragma unroll
    for (int mi = 0; mi < 4; ++mi) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float lm = -INFINITY;
#pragma unroll
            for (int ni = 0; ni < 8; ++ni)
                if (full || vl + 16 * ni < a.V) lm = fmaxf(lm, acc[mi][ni][r]);
            const float mx = row16_max(lm);
            float s = 0.f;
            int ix = 0x7fffffff;
            if (mx > -INFINITY) {
                const float mx2 = mx * LOG2E;  // exp(x - mx) = exp2(x log2e - mx log2e)
#pragma unroll
                for (int ni = 0; ni < 8; ++ni)
                    if (full || vl + 16 * ni < a.V) {
                        const float x = acc[mi][ni][r];
                        s += __builtin_amdgcn_exp2f(__builtin_fmaf(x, LOG2E, -mx2));
                        if (ARGMAX && x == mx) ix = min(ix, vl + 16 * ni);
                    }
            }
            s = row16_sum(s);
            if (ARGMAX) ix = row16_min(ix);
            if (l16 == 0) {
                const int row = 64 * wm + 16 * mi + 4 * g + r;
                sM[wn][row] = mx;
                sS[wn][row] = s;
                if (ARGMAX) sI[wn][row] = ix;
            }
        }
    }
    __syncthreads();
    if (tid < TM && r0 + tid < a.N) {
        const float m0 = sM[0][tid], m1 = sM[1][tid];
        const float m = fmaxf(m0, m1);
        float s = 0.f;
        if (m0 > -INFINITY) s += sS[0][tid] * __expf(m0 - m);
        if (m1 > -INFINITY) s += sS[1][tid] * __expf(m1 - m);
        const int64_t o = (int64_t)(r0 + tid) * p.n_vt + vt;
        p.part_m[o] = m;
        p.part_s[o] = s;
        if (ARGMAX) p.part_i[o] = (m1 > m0 || (m1 == m0 && sI[1][tid] < sI[0][tid])) ? sI[1][tid] : sI[0][tid];
    }
}

// backward G tile (256 rows x 256 vocab): recompute logits, write G^T [Vp][Rp]
// (and G [rows][Vp] when write_g)
__global__ void __launch_bounds__(WTHREADS) grad_tile_kernel(BwdParams p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ float sLse[TM], sScale[TM];
    __shared__ int sTgt[TM];
    const qpam_ce_bwd_args &a = p.a;
    const int n_rt = p.Rp / TM, n_vt = p.Vp / TN;
    const int item = xcd_item(blockIdx.x, n_rt * n_vt);
    if (item >= n_rt * n_vt) return;
    int rt, vt;
    big::grouped_tile(item, n_rt, n_vt, rt, vt);
    const int lr0 = rt * TM, v0 = vt * TN;
    const int tid = threadIdx.x;
    if (tid < TM) {
        const int lr = lr0 + tid, row = p.row0 + lr;
        float lse = 0.f, sc = 0.f;
        int tg = -1;
        if (lr < p.rows) {
            const int64_t t = a.targets[row];
            const bool valid = (t != a.ignore_index) && t >= 0 && t < a.V;
            lse = a.lse[row];
            sc = valid ? a.grad_scale[0] * (a.mask ? a.mask[row] : 1.f) : 0.f;
            tg = valid ? (int)t : -1;
        }
        sLse[tid] = lse;
        sScale[tid] = sc;
        sTgt[tid] = tg;
    }
    floatx4 acc[4][8];
    if constexpr (USE_DMA)
        wgemm_tile_dma((const U16 *)a.h + (int64_t)(p.row0 + lr0) * a.ldh, a.ldh, min(TM, p.rows - lr0),
                       (const U16 *)a.w + (int64_t)v0 * a.ldw, a.ldw, min(TN, a.V - v0), a.D, acc);
    else
        wgemm_tile((const U16 *)a.h + (int64_t)(p.row0 + lr0) * a.ldh, a.ldh, min(TM, p.rows - lr0),
                   (const U16 *)a.w + (int64_t)v0 * a.ldw, a.ldw, min(TN, a.V - v0), a.D, acc,
                   reinterpret_cast<U16 *>(smem_raw));
    const int w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
    U16 *G = (U16 *)p.gbuf;
    U16 *GT = (U16 *)p.gtbuf;
    // G^T rows (one per vocab entry) hold the tile's rows contiguously: each
    // 16-wide vocab slab of a wave's 64 x 128 tile goes through LDS so that it
    // leaves as 128-byte runs (the accumulator layout alone would write 32-byte
    // pieces).
    constexpr int GT_LD = 72;   // bf16 per staged vocab row: 64 tile rows + padding against bank conflicts
    __shared__ __align__(16) U16 sEpi[8 * 16 * GT_LD];
    U16 *tw = sEpi + w * 16 * GT_LD;
    // the 16 rows of this lane (rows 64 wm + 16 mi + 4 g + r) in registers: lse in
    // log2 units (exp(x - lse) = exp2(x log2e - lse log2e), one fma and one exp2),
    // +inf for rows without a gradient (their G is exp2(-inf) = 0), the scale and
    // the target column
    float hl[4][4], hs[4][4];
    int ht[4][4];
#pragma unroll
    for (int mi = 0; mi < 4; ++mi)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int rl = 64 * wm + 16 * mi + 4 * g + r;
            hs[mi][r] = sScale[rl];
            hl[mi][r] = hs[mi][r] != 0.f ? sLse[rl] * LOG2E : INFINITY;
            ht[mi][r] = sTgt[rl];
        }
    const bool full = v0 + TN <= a.V;  // every column of the tile is a vocabulary entry
#pragma unroll
    for (int ni = 0; ni < 8; ++ni) {
        const int vb = v0 + 128 * wn + 16 * ni, v = vb + l16;
        const bool vok = full || v < a.V;
#pragma unroll
        for (int mi = 0; mi < 4; ++mi) {
            const int rl0 = 64 * wm + 16 * mi + 4 * g;
            float x[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[mi][ni][r], LOG2E, -hl[mi][r]));
                x[r] = vok ? (e - (v == ht[mi][r] ? 1.f : 0.f)) * hs[mi][r] : 0.f;
            }
            const unsigned lo = pack_bf16x2(x[0], x[1]), hi = pack_bf16x2(x[2], x[3]);
            if (p.write_g) {
                const unsigned short gb[4] = {(unsigned short)(lo & 0xFFFFu), (unsigned short)(lo >> 16),
                                              (unsigned short)(hi & 0xFFFFu), (unsigned short)(hi >> 16)};
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (lr0 + rl0 + r < p.rows) G[(int64_t)(lr0 + rl0 + r) * p.Vp + v] = gb[r];
            }
            *reinterpret_cast<uint2 *>(tw + l16 * GT_LD + 16 * mi + 4 * g) = make_uint2(lo, hi);
        }
        // the slab is this wave's own: its LDS writes complete before its reads
        // (and the reads before the next slab's writes) without a block barrier
        wave_lds_sync();
        {   // lane -> (vocab row lane / 4, 16 tile rows (lane % 4) * 16 ..): 32 bytes each
            const int vl = lane >> 2, part = lane & 3;
            const uint4 *src = reinterpret_cast<const uint4 *>(tw + vl * GT_LD + 16 * part);
            const uint4 d0 = src[0], d1 = src[1];
            uint4 *dst = reinterpret_cast<uint4 *>(GT + (int64_t)(vb + vl) * p.Rp + lr0 + 64 * wm + 16 * part);
            dst[0] = d0;
            dst[1] = d1;
        }
        wave_lds_sync();
    }
}
}  // namespace wide

// Token scores' bf16 tiles, 256 x 256: loads, swizzle and wave layout as in `wide`, with a
// k-step's first fragments read from LDS between the MFMAs of the step before, so that no
// wave waits for LDS at the head of a step.  16384 x 50261 x 1024: scores 1.55 ms (1.09
// PFLOP/s, the MFMA pipes about 55 % busy at the 1.9 GHz that the card holds under this load, LDS
// 23 %), G^T 1.78 ms with 1.65 GB of stores; two blocks of 128 x 256 a CU took 1.85 and 2.11.
namespace tiles {
constexpr int TM = wide::TM, TN = wide::TN, DK = wide::DK, TT = wide::WTHREADS;
using U16 = unsigned short;

struct Stage {
    U16 a[TM * DK], b[TN * DK];
};
// The wave's share of a tile is 64 rows x 16 NI columns; NI = 8 is the whole tile.
template <int NI> struct Frags {
    bf16x8 a[4], b[NI / 2];  // the step's A fragments and the first half of its B fragments
};
// A wave's four loads of a stage (16 rows of 64 bytes each, two of A and two of B): a
// uniform base that advances and 32-bit offsets that stay (row strides below 2^22).
struct Loads {
    const char *a, *b;
    unsigned ao[2], bo[2];
};

__device__ __forceinline__ void to_lds(const char *from, U16 *lds) {
    __builtin_amdgcn_global_load_lds(reinterpret_cast<const unsigned *>(from), reinterpret_cast<unsigned *>(lds), 16, 0, 0);
}
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

__device__ __forceinline__ void load(Stage &s, const Loads &q, int step) {
    const int w = wave_id();
    const char *a = q.a + (int64_t)step * (2 * DK), *b = q.b + (int64_t)step * (2 * DK);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        to_lds(a + q.ao[j], &s.a[(32 * w + 16 * j) * DK]);
        to_lds(b + q.bo[j], &s.b[(32 * w + 16 * j) * DK]);
    }
}

__device__ __forceinline__ bf16x8 fragment(const U16 *at, int i) {
    return *reinterpret_cast<const bf16x8 *>(at + 16 * i * DK);
}

// The products of a step: the second half of its B fragments is read in front of the
// products of the first, the next step's first fragments (stage s) between those of the second.
template <int NI>
__device__ __forceinline__ void step(const Frags<NI> &cur, const Stage &c, Frags<NI> &next, const Stage &s,
                                     floatx4 (&acc)[4][NI], int aat, int bat) {
    constexpr int H = NI / 2;
    bf16x8 late[H];
#pragma unroll
    for (int i = 0; i < H; ++i) late[i] = fragment(c.b + bat, H + i);
#pragma unroll
    for (int ni = 0; ni < H; ++ni)
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
            acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cur.a[mi], cur.b[ni], acc[mi][ni], 0, 0, 0);
#pragma unroll
    for (int ni = 0; ni < H; ++ni)
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
            acc[mi][H + ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cur.a[mi], late[ni], acc[mi][H + ni], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        next.a[i] = fragment(s.a + aat, i);
        if (i < H) next.b[i < H ? i : 0] = fragment(s.b + bat, i);
    }
    if constexpr (NI < 8) return;
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);   // LDS reads
    __builtin_amdgcn_sched_group_barrier(0x008, 16, 0);  // MFMAs
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) {
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
}

// A block takes tile after tile (one block a CU): the first three stages of the next tile
// are loaded while this one is in its epilogue.  Tiles in the order and by the XCD ranges
// of big::xcd_item / grouped_tile.
struct Walk {
    int item, end, n_rt, n_vt, rt, vt;
    __device__ __forceinline__ Walk(int rts, int vts) : n_rt(rts), n_vt(vts) {
        const int total = n_rt * n_vt, per = (total + big::XCDS - 1) / big::XCDS, x = blockIdx.x % big::XCDS;
        item = x * per + blockIdx.x / big::XCDS;
        end = min(total, (x + 1) * per);
        place();
    }
    __device__ __forceinline__ bool more() const { return item < end; }
    __device__ __forceinline__ void place() {
        if (more()) big::grouped_tile(item, n_rt, n_vt, rt, vt);
    }
    __device__ __forceinline__ void next() {
        item += gridDim.x / big::XCDS;
        place();
    }
};
// blocks of a launch: every XCD's 32 CUs, or one block a tile if there are fewer
inline int grid(int tiles) { return big::XCDS * std::min(32, (tiles + big::XCDS - 1) / big::XCDS); }

struct Stages {
    Stage &s0, &s1, &s2, &s3;
};

// Rows past the end of an operand re-read its last row.
__device__ __forceinline__ Loads loads(const U16 *A, int64_t lda, int a_rows, const U16 *B, int64_t ldb, int b_rows) {
    const int w = wave_id(), lane = threadIdx.x & 63;
    Loads q{reinterpret_cast<const char *>(A), reinterpret_cast<const char *>(B), {}, {}};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = 32 * w + 16 * j + (lane >> 2), c = 16 * wide::swz(row, lane & 3);
        q.ao[j] = 2u * (unsigned)min(row, a_rows - 1) * (unsigned)lda + c;
        q.bo[j] = 2u * (unsigned)min(row, b_rows - 1) * (unsigned)ldb + c;
    }
    return q;
}
__device__ __forceinline__ void start(const Stages &s, const Loads &q, int KT) {
    load(s.s0, q, 0);
    load(s.s1, q, min(1, KT - 1));
    load(s.s2, q, min(2, KT - 1));
}

// The product whose first stages start() has under way: acc[mi][ni] lane holds
// C[64*(w>>1) + 16mi + 4g + r][16*NI*(w&1) + 16ni + l16].  Step kt multiplies stage kt, reads
// the first fragments of stage kt + 1 and starts the loads of stage kt + 3, four a wave
// (past the end they re-read the last step): at its end "stage kt + 2 landed" is vmcnt
// <= 4.  The stages are free and no load is in flight when it returns.
template <int NI>
__device__ __forceinline__ void product(const Stages &st, const Loads &q, int KT, floatx4 (&acc)[4][NI]) {
    Stage &s0 = st.s0, &s1 = st.s1, &s2 = st.s2, &s3 = st.s3;
    const int tid = threadIdx.x, w = wave_id(), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
#pragma unroll
    for (int mi = 0; mi < 4; ++mi)
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = floatx4{0.f, 0.f, 0.f, 0.f};
    // fragment (row, chunk g); the swizzle repeats every eight rows
    const int aat = (64 * (w >> 1) + l16) * DK + 8 * wide::swz(l16, g);
    const int bat = (16 * NI * (w & 1) + l16) * DK + 8 * wide::swz(l16, g);
    stage_barrier<4>();
    Frags<NI> f0, f1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f0.a[i] = fragment(s0.a + aat, i);
        if (i < NI / 2) f0.b[i < NI / 2 ? i : 0] = fragment(s0.b + bat, i);
    }
#define QPAM_STEP(KT_, CUR, STAGE, NEXT, NEXT_STAGE, FREE)                                     \
    load(FREE, q, min((KT_) + 3, KT - 1));                                                     \
    step(CUR, STAGE, NEXT, NEXT_STAGE, acc, aat, bat);                                         \
    stage_barrier<4>();
    int kt = 0;
    for (; kt + 3 < KT; kt += 4) {
        QPAM_STEP(kt, f0, s0, f1, s1, s3)
        QPAM_STEP(kt + 1, f1, s1, f0, s2, s0)
        QPAM_STEP(kt + 2, f0, s2, f1, s3, s1)
        QPAM_STEP(kt + 3, f1, s3, f0, s0, s2)
    }
    if (kt < KT) { QPAM_STEP(kt, f0, s0, f1, s1, s3) }
    if (kt + 1 < KT) { QPAM_STEP(kt + 1, f1, s1, f0, s2, s0) }
    if (kt + 2 < KT) { QPAM_STEP(kt + 2, f0, s2, f1, s3, s1) }
#undef QPAM_STEP
    stage_barrier<0>();
}

// The block's LDS writes before it are read after it; loads and stores stay in flight.
__device__ __forceinline__ void block_lds_sync() {
    wide::wave_lds_sync();
    __builtin_amdgcn_s_barrier();
    wave_lds_order();
}

// The tokens of a tile's rows, and the rows (a bit each, 64 a word) whose token is one of its
// columns: about one row of the 256 where tokens are spread, so most groups of 16 rows skip
// the search for it (searched for in every group the scores take 2 % longer).
struct Tokens {
    int of[TM];
    uint64_t here[TM / 64];
};

// A tile's (m, s, t) per row: over each wave's columns from v0 on, then the two waves of a row.
template <int NI>
__device__ __forceinline__ void reduce_rows(const FwdParams &p, const floatx4 (&acc)[4][NI], int r0, int v0, int vt,
                                            float (&sM)[2][TM], float (&sS)[2][TM], float (&sT)[2][TM], const Tokens &tokens) {
    const qpam_ce_fwd_args &a = p.a;
    const int tid = threadIdx.x, w = wave_id(), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
    const int vl = v0 + 16 * NI * wn + l16;  // this lane's column in tile ni: vl + 16 ni
    wave_lds_order();                        // the tokens, written in front of the product's barriers
    const uint64_t here = tokens.here[wm];
    const uint32_t here_lo = __builtin_amdgcn_readfirstlane((int)here), here_hi = __builtin_amdgcn_readfirstlane((int)(here >> 32));
    auto rows = [&](auto whole) {            // whole: no column past the vocabulary
#pragma unroll
        for (int mi = 0; mi < 4; ++mi) {
            if (((mi < 2 ? here_lo : here_hi) >> (16 * (mi & 1))) & 0xFFFF) {
                const intx4 token = *reinterpret_cast<const intx4 *>(&tokens.of[64 * wm + 16 * mi + 4 * g]);
#pragma unroll
                for (int r = 0; r < 4; ++r) keep_token(p, acc[mi], r, r0 + 64 * wm + 16 * mi + 4 * g + r, token[r], vl);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float mx = -INFINITY;
#pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                    if (whole || vl + 16 * ni < a.V) mx = fmaxf(mx, acc[mi][ni][r]);
                const float m = row16_max(mx);
                float s = 0.f, t = 0.f;
#pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                    if (whole || vl + 16 * ni < a.V) {
                        const float d = acc[mi][ni][r] - m, e = __builtin_amdgcn_exp2f(d * p.c);
                        s += e;
                        t = __builtin_fmaf(e, d, t);
                    }
                s = row16_sum(s);
                t = row16_sum(t);
                if (l16 == 0) {
                    const int row = 64 * wm + 16 * mi + 4 * g + r;
                    sM[wn][row] = m;
                    sS[wn][row] = s;
                    sT[wn][row] = t * p.c;
                }
            }
        }
    };
    if (v0 + 32 * NI <= a.V) rows(std::true_type{});
    else rows(std::false_type{});
    block_lds_sync();
    if (tid < TM && r0 + tid < a.N) {
        float m = sM[0][tid], s = sS[0][tid], t = sT[0][tid];
        join_scores(p.c, m, s, t, sM[1][tid], sS[1][tid], sT[1][tid]);
        const int64_t o = (int64_t)(r0 + tid) * p.n_vt + vt;
        p.part_m[o] = m;
        p.part_s[o] = s;
        p.part_t[o] = t;
    }
}

// The vocabulary's columns: `full` tiles of 256 that fill whole rounds of the 256 CUs, the
// rest (what would be a last round with few blocks) in tiles of 32 NARROW columns, one a
// block, if they fit one round.
struct Columns {
    int full, narrow, n_vt;  // narrow: 2 (64 columns) or 4 (128)
};
inline Columns columns(int N, int V) {
    const int64_t n_rt = (N + TM - 1) / TM, n_ct = (V + TN - 1) / TN;
    const int64_t full = n_rt * n_ct / 256 * 256 / n_rt, rest = V - full * TN;
    if (rest > 0)
        for (int ni = 2; ni <= 4; ni *= 2) {
            const int64_t more = (rest + 32 * ni - 1) / (32 * ni);
            if (n_rt * more <= 256) return {(int)full, ni, (int)(full + more)};
        }
    return {(int)n_ct, 2, (int)n_ct};
}

template <int NARROW>
__global__ void __launch_bounds__(TT) scores_tile_kernel(FwdParams p) {
    __shared__ __align__(16) Stage s0, s1, s2, s3;
    __shared__ float sM[2][TM], sS[2][TM], sT[2][TM];
    __shared__ __align__(16) Tokens sTokens[2];  // of this tile and the next
    const qpam_ce_fwd_args &a = p.a;
    const Stages stages{s0, s1, s2, s3};
    const int KT = a.D / DK, n_rt = (a.N + TM - 1) / TM, tid = threadIdx.x;
    Walk at(n_rt, p.full_vt);
    const bool last = (int)blockIdx.x < n_rt * (p.n_vt - p.full_vt);
    const int last_rt = blockIdx.x % n_rt, last_ct = blockIdx.x / n_rt;
    const int last_v0 = p.full_vt * TN + 32 * NARROW * last_ct;
    Loads q;
    struct Place {
        int r0, v0, cols;
    };
    auto place = [&]() { return at.more() ? Place{at.rt * TM, at.vt * TN, TN} : Place{last_rt * TM, last_v0, 32 * NARROW}; };
    auto load_next = [&]() {
        if (!at.more() && !last) return;
        const Place t = place();
        q = loads((const U16 *)a.h + (int64_t)t.r0 * a.ldh, a.ldh, min(TM, a.N - t.r0), (const U16 *)a.w + (int64_t)t.v0 * a.ldw,
                  a.ldw, min(t.cols, a.V - t.v0));
        start(stages, q, KT);
    };
    // the id of this thread's row in the tile at place(), loaded in front of the product before it
    auto load_id = [&]() { return a.targets[min(place().r0 + (tid & (TM - 1)), a.N - 1)]; };
    auto put_tokens = [&](int64_t id, int buf) {
        if (tid >= TM) return;
        const Place t = place();
        const int token = t.r0 + tid < a.N ? token_of(p, id) : -1;
        const uint64_t here = __ballot(token >= t.v0 && token - t.v0 < t.cols);
        sTokens[buf].of[tid] = token;
        if ((tid & 63) == 0) sTokens[buf].here[wave_id()] = here;
    };
    put_tokens(load_id(), 0);
    load_next();
    int buf = 0;
    while (at.more()) {
        const int rt = at.rt, vt = at.vt;
        at.next();
        const int64_t id = load_id();
        floatx4 acc[4][8];
        product(stages, q, KT, acc);
        put_tokens(id, buf ^ 1);
        load_next();
        reduce_rows(p, acc, rt * TM, vt * TN, vt, sM, sS, sT, sTokens[buf]);
        buf ^= 1;
    }
    if (!last) return;
    floatx4 acc[4][NARROW];
    product(stages, q, KT, acc);
    reduce_rows(p, acc, last_rt * TM, last_v0, p.full_vt + last_ct, sM, sS, sT, sTokens[buf]);
}

// G^T [Vp][Rp] without the tokens' one-hot terms; zero past the vocabulary and past the rows.
// Tiles as in the scores' kernel.
template <int NARROW>
__global__ void __launch_bounds__(TT) scores_grad_kernel(BwdParams p) {
    constexpr int LD = 72;  // bf16 per staged vocab row: 64 tile rows + padding against bank conflicts
    __shared__ __align__(16) Stage s0, s1, s2, s3;
    __shared__ __align__(16) U16 sSlab[8 * 16 * LD];
    __shared__ __align__(16) float sRow[2][3][TM];  // the rows' scores, of this tile and the next
    const qpam_ce_bwd_args &a = p.a;
    const Stages stages{s0, s1, s2, s3};
    const int KT = a.D / DK, n_rt = p.Rp / TM;
    const int tid = threadIdx.x, w = wave_id(), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wm = w >> 1, wn = w & 1;
    Walk at(n_rt, p.full_vt);
    const bool last = (int)blockIdx.x < n_rt * ((p.Vp - p.full_vt * TN) / (32 * NARROW));
    const int last_rt = blockIdx.x % n_rt, last_v0 = p.full_vt * TN + 32 * NARROW * (blockIdx.x / n_rt);
    U16 *GT = (U16 *)p.gtbuf;
    U16 *slab = sSlab + w * 16 * LD;
    // a slab's way out in two stores of eight whole 128-byte lines: vocab rows lane / 8 and
    // lane / 8 + 8, 16 bytes a lane
    const U16 *from = slab + (lane >> 3) * LD + 8 * (lane & 7);
    const unsigned to = 2u * ((lane >> 3) * (unsigned)p.Rp + 8 * (lane & 7));
    Loads q;
    auto load_next = [&](int buf) {
        if (!at.more() && !last) return;
        const int rt = at.more() ? at.rt : last_rt, v0 = at.more() ? at.vt * TN : last_v0, lr0 = rt * TM;
        const RowScore x = row_score(p, lr0 + (tid & (TM - 1)));
        if (tid < TM) {
            sRow[buf][0][tid] = x.m;
            sRow[buf][1][tid] = x.base;
            sRow[buf][2][tid] = x.slope;
        }
        const int vr = min(v0, a.V - 1);  // a narrow tile of padding alone reads the last row
        q = loads((const U16 *)a.h + (int64_t)(p.row0 + lr0) * a.ldh, a.ldh, min(TM, p.rows - lr0), (const U16 *)a.w + (int64_t)vr * a.ldw,
                  a.ldw, min(at.more() ? TN : 32 * NARROW, a.V - vr));
        start(stages, q, KT);
    };
    // A 16-wide vocab slab of a wave goes through LDS and leaves as 128-byte runs of G^T.
    auto write = [&](const auto &acc, auto ni_count, int lr0, int v0, int buf) {
        constexpr int NI = decltype(ni_count)::value;
        // this lane's rows are 64 wm + 16 mi + 4 g + r; their scores are read again for every
        // slab, as 48 registers of them beside the accumulators spill
        const float *mine = &sRow[buf][0][64 * wm + 4 * g];
        auto slabs = [&](auto whole) {  // whole: every column is a vocabulary entry, every row a row
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                const int vb = v0 + 16 * NI * wn + 16 * ni, v = vb + l16;
#pragma unroll
                for (int mi = 0; mi < 4; ++mi) {
                    const int rl0 = 64 * wm + 16 * mi + 4 * g;
                    const floatx4 hm = *reinterpret_cast<const floatx4 *>(mine + 16 * mi);
                    const floatx4 h0 = *reinterpret_cast<const floatx4 *>(mine + TM + 16 * mi);
                    const floatx4 h1 = *reinterpret_cast<const floatx4 *>(mine + 2 * TM + 16 * mi);
                    float x[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float u = score_u(acc[mi][ni][r], hm[r], p.c);
                        x[r] = __builtin_amdgcn_exp2f(u) * __builtin_fmaf(h1[r], u, h0[r]);
                        if (!whole && (v >= a.V || lr0 + rl0 + r >= p.rows)) x[r] = 0.f;
                    }
                    const unsigned lo = pack_bf16x2(x[0], x[1]), hi = pack_bf16x2(x[2], x[3]);
                    *reinterpret_cast<uint2 *>(slab + l16 * LD + 16 * mi + 4 * g) = make_uint2(lo, hi);
                }
                wave_lds_order();  // the slab is this wave's own, and a wave's LDS accesses stay in order
                const uint4 d0 = *reinterpret_cast<const uint4 *>(from), d1 = *reinterpret_cast<const uint4 *>(from + 8 * LD);
                char *out = reinterpret_cast<char *>(GT + (int64_t)vb * p.Rp + lr0 + 64 * wm);
                *reinterpret_cast<uint4 *>(out + to) = d0;
                *reinterpret_cast<uint4 *>(out + 16ll * p.Rp + to) = d1;
                wave_lds_order();
            }
        };
        if (v0 + 32 * NI <= a.V && lr0 + TM <= p.rows) slabs(std::true_type{});
        else slabs(std::false_type{});
    };
    load_next(0);
    int buf = 0;
    for (; at.more(); buf ^= 1) {
        floatx4 acc[4][8];
        product(stages, q, KT, acc);
        const int lr0 = at.rt * TM, v0 = at.vt * TN;
        at.next();
        load_next(buf ^ 1);
        write(acc, std::integral_constant<int, 8>{}, lr0, v0, buf);
    }
    if (!last) return;
    floatx4 acc[4][NARROW];
    product(stages, q, KT, acc);
    write(acc, std::integral_constant<int, NARROW>{}, last_rt * TM, last_v0, buf);
}
// dH = (G^T)^T W (AT) and dW = G^T H, [M][N] = A B with A [K][M] or [M][K] and B [b_rows][N] as
// they stand (b_rows <= K, A is zero past them).  A stage of an operand whose rows are k
// holds 32 of them by 256 columns, its 32-byte pieces swizzled by h(row) so that the eight
// rows that half a wave's transpose read takes are in distinct banks.  K in `ranges` ranges
// of kper where tiles are few; tiles in the order range, M, N over the XCDs' block ranges, so
// that those which share operands share an L2.  A range's sums leave in fp32, each in its
// place of `out`.
// The entries of G at the rows' tokens come in fp32 beside it (TokenTerms): dH's tiles add
// g W[id] to their rows at the end; dW's tiles look for their own tokens among the rows' ids
// and multiply them as further steps of 32 rows, g in three bf16 parts.  A range of K has the
// entries that lie in it.
// Against 50261 x 768, dH with the sum: 16 rows 29 us, 200 rows 39, bound by reading W and
// the partial sums (hipBLASLt, with 20 and 51 blocks: 107 and 197).  16384 rows, 50261 x
// 1024: dW 1.40 ms, dH 1.43, 1.19 PFLOP/s (hipBLASLt 1.60 and 1.51); the tokens' entries take 5 us of
// a call of few rows, 0.4 % of this one.
__device__ __forceinline__ int h_of(int row) { return (row & 3) | ((row >> 3) & 1) << 2; }

enum { OUT_BF16, OUT_F32, OUT_ADD };

// dH: of rows 0 .. M - 1; dW: of rows 0 .. b_rows - 1, with row 0 of the product vocabulary entry v0.
// Both arrays 16-byte aligned and a multiple of four long.
struct TokenTerms {
    const float *g;
    const int *id;  // -1: none
    int v0;
};
constexpr int SCAN = 16 * TT;  // rows whose ids a block looks through at once

template <bool AT>
__global__ void __launch_bounds__(TT) gemm_kernel(const U16 *A, int64_t lda, int M, const U16 *B, int64_t ldb, int b_rows, int N, int K,
                                                  int kper, int ranges, void *out, int64_t ldo, int64_t range_stride, int mode,
                                                  TokenTerms t) {
    __shared__ __align__(16) Stage s0, s1, s2, s3;
    const int n_ct = (N + TN - 1) / TN, tiles = (M + TM - 1) / TM * n_ct;
    const int item = big::xcd_item(blockIdx.x, tiles * ranges);
    if (item >= tiles * ranges) return;
    const int z = item / tiles, rt = (item - z * tiles) / n_ct, ct = item - z * tiles - rt * n_ct;
    const int m0 = rt * TM, n0 = ct * TN, k0 = z * kper, KT = min(kper, K - k0) / DK;
    const int w = wave_id(), lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    // a wave's load j: rows 4 w + 2 j and the next, a 16-byte chunk a lane
    int row[2];
    unsigned ao[2], bo[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        row[j] = 4 * w + 2 * j + (lane >> 5);
        const int col = 16 * (((lane >> 1) & 15) ^ h_of(row[j])) + 8 * (lane & 1);
        bo[j] = 2u * min(col, N - n0 - 8);
        const int arow = 32 * w + 16 * j + (lane >> 2);  // A [M][K]: 16 rows of 64 bytes, every row of a tile in memory
        ao[j] = AT ? 2u * ((unsigned)row[j] * (unsigned)lda + col) : 2u * (unsigned)arow * (unsigned)lda + 16 * wide::swz(arow, lane & 3);
    }
    const U16 *a0 = AT ? A + (int64_t)k0 * lda + m0 : A + (int64_t)m0 * lda + k0;
    auto load = [&](Stage &s, int step) {
        const int k = k0 + step * DK, b0 = min(k, b_rows - 1);  // past B's rows A is zero: its last row again
        const char *a = reinterpret_cast<const char *>(a0 + (AT ? (int64_t)step * DK * lda : (int64_t)step * DK));
        const char *b = reinterpret_cast<const char *>(B + (int64_t)b0 * ldb + n0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            to_lds(a + ao[j], &s.a[AT ? (4 * w + 2 * j) * TM : (32 * w + 16 * j) * DK]);
            to_lds(b + (2u * (unsigned)min(row[j], b_rows - 1 - b0) * (unsigned)ldb + bo[j]), &s.b[(4 * w + 2 * j) * TN]);
        }
    };
    // column l16 of a 16-column chunk, k = 8 g ..: rows 8 g + l16 / 4 and four behind it
    const int frow = 8 * g + (l16 >> 2), at0 = frow * TM + 16 * h_of(frow) + 4 * (l16 & 3);
    const int a_at = (64 * (w >> 1) + l16) * DK + 8 * wide::swz(l16, g);
    auto fragment_t = [&](const U16 *s, int base, int c) {  // chunk c, swizzled: c ^ h(row)
        const U16 *at = s + (base ^ (16 * c));
        const shortx4 lo = lds_read_tr(at), hi = lds_read_tr(at + 4 * TM);
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    floatx4 acc[4][8];
#pragma unroll
    for (int mi = 0; mi < 4; ++mi)
#pragma unroll
        for (int ni = 0; ni < 8; ++ni) acc[mi][ni] = floatx4{0.f, 0.f, 0.f, 0.f};
    // the stage after this one is in LDS, and every wave is done reading this one
    auto landed = [&]() {
        stage_barrier<8>();
        wave_lds_order();
    };
    load(s0, 0);
    load(s1, min(1, KT - 1));
    load(s2, min(2, KT - 1));
    landed();
    auto step = [&](int kt, const Stage &s, Stage &free) {  // stage kt; kt + 3 into the stage that kt - 1 left
        load(free, min(kt + 3, KT - 1));
        int base = at0;
        asm volatile("" : "+v"(base));  // the fragments' addresses are made here: kept over the steps they spill
        bf16x8 a[4], b[4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (half == 0) a[i] = AT ? fragment_t(s.a, base, 4 * (w >> 1) + i) : fragment(s.a + a_at, i);
                b[i] = fragment_t(s.b, base, 8 * (w & 1) + 4 * half + i);
            }
#pragma unroll
            for (int ni = 0; ni < 4; ++ni)
#pragma unroll
                for (int mi = 0; mi < 4; ++mi)
                    acc[mi][4 * half + ni] =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[mi], b[ni], acc[mi][4 * half + ni], 0, 0, 0);
        }
        landed();
    };
    int kt = 0;
    for (; kt + 3 < KT; kt += 4) {
        step(kt, s0, s3);
        step(kt + 1, s1, s0);
        step(kt + 2, s2, s1);
        step(kt + 3, s3, s2);
    }
    if (kt < KT) step(kt, s0, s3);
    if (kt + 1 < KT) step(kt + 1, s1, s0);
    if (kt + 2 < KT) step(kt + 2, s2, s1);
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // no direct load outlives the wave
    const int m1 = m0 + 64 * (w >> 1) + 4 * g, n1 = n0 + 128 * (w & 1) + l16;
    if constexpr (AT) {  // g W[id], the columns of four rows in flight
#pragma unroll
        for (int mi = 0; mi < 4; ++mi) {
            const int m = m1 + 16 * mi;
            const intx4 id = m < M ? *reinterpret_cast<const intx4 *>(t.id + m) : intx4{-1, -1, -1, -1};
            const floatx4 gt = m < M ? *reinterpret_cast<const floatx4 *>(t.g + m) : floatx4{0.f, 0.f, 0.f, 0.f};
            bool on[4], any = false;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                on[r] = m + r < M && id[r] >= k0 && id[r] < k0 + kper;
                any |= on[r];
            }
            if (__ballot(any) == 0) continue;
            U16 x[4][8];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int ni = 0; ni < 8; ++ni) x[r][ni] = B[(int64_t)(on[r] ? id[r] : 0) * ldb + min(n1 + 16 * ni, N - 1)];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int ni = 0; ni < 8; ++ni)
                    acc[mi][ni][r] = on[r] ? __builtin_fmaf(gt[r], bf16_to_f32(x[r][ni]), acc[mi][ni][r]) : acc[mi][ni][r];
        }
    } else {
        // the stages' memory: g's parts as A tiles in s0.a, s1.a and s3.a, H's rows in s0.b, the list of
        // matches (row in the scan << 8 | vocabulary entry in the tile) over s2, the waves' counts in s1.b
        U16 *const part[3] = {s3.a, s1.a, s0.a};  // smallest first
        int *list = reinterpret_cast<int *>(&s2), *counts = reinterpret_cast<int *>(s1.b);
        const int tid = threadIdx.x, v0 = t.v0 + m0, k1 = min(k0 + kper, b_rows);
        for (int c0 = k0; c0 < k1; c0 += SCAN) {
            uint32_t hits = 0;
            int v[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = c0 + 16 * tid + 4 * q;
                const intx4 id = row < k1 ? *reinterpret_cast<const intx4 *>(t.id + row) : intx4{-1, -1, -1, -1};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[4 * q + i] = id[i] - v0;
                    if (row + i < k1 && id[i] >= v0 && v[4 * q + i] < TM) hits |= 1u << (4 * q + i);
                }
            }
            int before = __popc(hits);  // inclusive over the wave's lanes
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(before, off);
                if (lane >= off) before += o;
            }
            __syncthreads();  // the products and the list of the scan before are done with
            if (lane == 63) counts[w] = before;
            __syncthreads();
            int total = 0, at = before - __popc(hits);
            for (int x = 0; x < TT / 64; ++x) {
                if (x < w) at += counts[x];
                total += counts[x];
            }
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (hits >> i & 1) list[at++] = (16 * tid + i) << 8 | v[i];
            for (int e0 = 0; e0 < total; e0 += DK) {
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 3; ++i)
#pragma unroll
                    for (int j = 0; j < TM * DK / 8 / TT; ++j)
                        reinterpret_cast<uint4 *>(part[i])[tid + j * TT] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int from = c0 + (list[min(e0 + row[j], total - 1)] >> 8);
                    to_lds(reinterpret_cast<const char *>(B + (int64_t)from * ldb + n0) + bo[j], &s0.b[(4 * w + 2 * j) * TN]);
                }
                __syncthreads();
                if (tid < DK && e0 + tid < total) {
                    const int e = list[e0 + tid], vl = e & 255;
                    float x = t.g[c0 + (e >> 8)];
#pragma unroll
                    for (int i = 2; i >= 0; --i) {
                        const U16 b = __builtin_bit_cast(U16, (__bf16)x);
                        part[i][vl * DK + 8 * wide::swz(vl, tid >> 3) + (tid & 7)] = b;
                        x -= bf16_to_f32(b);
                    }
                }
                __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
                __syncthreads();
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    bf16x8 b[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[i] = fragment_t(s0.b, at0, 8 * (w & 1) + 4 * half + i);
#pragma unroll
                    for (int i = 0; i < 3; ++i)
#pragma unroll
                        for (int mi = 0; mi < 4; ++mi) {
                            const bf16x8 a = fragment(part[i] + a_at, mi);
#pragma unroll
                            for (int ni = 0; ni < 4; ++ni)
                                acc[mi][4 * half + ni] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[ni], acc[mi][4 * half + ni], 0, 0, 0);
                        }
                }
            }
        }
    }
    const int64_t first = z * range_stride + (int64_t)m1 * ldo + n1;
    auto store = [&](auto *to, auto add) {  // to: the lane's first element
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (m1 + 16 * mi + r < M) {
#pragma unroll
                    for (int ni = 0; ni < 8; ++ni)
                        if (n1 + 16 * ni < N) {
                            if constexpr (sizeof(*to) == 2) to[16 * ni] = __builtin_bit_cast(U16, (__bf16)acc[mi][ni][r]);
                            else to[16 * ni] = add ? to[16 * ni] + acc[mi][ni][r] : acc[mi][ni][r];
                        }
                }
                to += r < 3 ? ldo : 13 * ldo;
            }
    };
    if (mode == OUT_BF16) store(static_cast<U16 *>(out) + first, std::false_type{});
    else if (mode == OUT_F32) store(static_cast<float *>(out) + first, std::false_type{});
    else store(static_cast<float *>(out) + first, std::true_type{});
}
}  // namespace tiles

// Token scores of few rows (a decode step's), bound by reading the table once.  A wave
// takes 16 table rows and every hidden row, 16 MI of them.  The table streams global ->
// LDS by direct loads in stages of 128 bytes a row, three stages deep, each wave its own
// rows (no barrier); the hidden rows in stages of 256 bytes a row, two deep, shared by
// the block.  Both are XOR-swizzled by 16-byte chunks so that the 16 rows of a fragment
// read distinct banks, and both operands take a lane's 16 bytes as consecutive k.
// Measured on 50261 x 1536 bf16 (154 MB): a load instruction has to cover whole 128-byte
// lines (16 rows x 64 bytes straight to registers: 45 us), and 197 blocks of 16 waves
// balance the CUs better than 786 of 4 (35 us).
namespace thin {
constexpr int ROWS = 64;                     // at most this many hidden rows
constexpr int WB = 128, HB = 256;            // bytes a row of a table / hidden stage
__host__ __device__ constexpr int waves(int V) { return V > 64 * 512 ? 16 : 4; }  // two blocks of 4 waves a CU, then 16

__device__ __forceinline__ void mma(uintx4 w, uintx4 h, floatx4 &acc, unsigned short) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, h), acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(uintx4 w, uintx4 h, floatx4 &acc, float) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[i]), __uint_as_float(h[i]), acc, 0, 0, 0);
}
__device__ __forceinline__ void to_lds(const char *from, char *lds) {
    __builtin_amdgcn_global_load_lds(reinterpret_cast<const unsigned *>(from), reinterpret_cast<unsigned *>(lds), 16, 0, 0);
}
// direct loads still in flight at most `n`, the wave's LDS reads are done and later ones stay behind the wait
template <int N> __device__ __forceinline__ void landed() {
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(N) & ~0xF00);
    wave_lds_order();
}

template <typename T, int MI, int NW>
__global__ void __launch_bounds__(64 * NW) scores_kernel(FwdParams p) {
    __shared__ __align__(16) char sW0[NW * 16 * WB], sW1[NW * 16 * WB], sW2[NW * 16 * WB];
    __shared__ __align__(16) char sH0[16 * MI * HB], sH1[16 * MI * HB];
    __shared__ float sM[NW][16 * MI], sS[NW][16 * MI], sT[NW][16 * MI];
    constexpr int HI = MI * 4 / NW > 0 ? MI * 4 / NW : 1;  // hidden-stage loads of a wave (spare waves repeat one)
    const qpam_ce_fwd_args &a = p.a;
    const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int v0 = (blockIdx.x * NW + w) * 16;
    int token[MI];  // of the lane's hidden rows
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) token[mi] = row_token(p, 16 * mi + l16);
    const int bytes = a.D * (int)sizeof(T), steps = bytes / 64, chunks = (bytes + HB - 1) / HB;
    // Rows past the end of an operand re-read its last row, chunks past a row's end its last
    // chunk.  A table load covers 8 rows, a hidden load 4; lane -> (row, chunk ^ row).
    const char *wrow[2], *hrow[HI];
    int hc[HI];
    const int wc = 16 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
    for (int i = 0; i < 2; ++i)
        wrow[i] = reinterpret_cast<const char *>((const T *)a.w + (int64_t)min(v0 + 8 * i + (lane >> 3), a.V - 1) * a.ldw);
#pragma unroll
    for (int i = 0; i < HI; ++i) {
        const int row = ((w * HI + i) % (4 * MI)) * 4 + (lane >> 4);
        hrow[i] = reinterpret_cast<const char *>((const T *)a.h + (int64_t)min(row, a.N - 1) * a.ldh);
        hc[i] = 16 * ((lane & 15) ^ (row & 15));
    }
    auto load_w = [&](char *lds, int stage) {
#pragma unroll
        for (int i = 0; i < 2; ++i) to_lds(wrow[i] + min(stage * WB + wc, bytes - 16), lds + (w * 16 + 8 * i) * WB);
    };
    auto load_h = [&](char *lds, int chunk) {
#pragma unroll
        for (int i = 0; i < HI; ++i)
            to_lds(hrow[i] + min(chunk * HB + hc[i], bytes - 16), lds + ((w * HI + i) % (4 * MI)) * 4 * HB);
    };
    floatx4 acc[MI];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) acc[mi] = floatx4{0.f, 0.f, 0.f, 0.f};
    // one table stage (two 64-byte steps) against half a hidden stage
    auto multiply = [&](const char *sw, const char *sh, int stage) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            if (2 * stage + q < steps) {
                const uintx4 x = *reinterpret_cast<const uintx4 *>(sw + (w * 16 + l16) * WB + 16 * ((4 * q + g) ^ (l16 & 7)));
#pragma unroll
                for (int mi = 0; mi < MI; ++mi)
                    mma(x, *reinterpret_cast<const uintx4 *>(sh + (16 * mi + l16) * HB + 16 * ((8 * (stage & 1) + 4 * q + g) ^ l16)),
                        acc[mi], T());
            }
        }
    };
    // Loads leave in the order W(0) W(1) h(0) | h(j+1) W(2j+2) .. W(2j+3) .. of chunk j, two a
    // table stage; every wave issues the same number, past the end too.
    load_w(sW0, 0);
    load_w(sW1, 1);
    load_h(sH0, 0);
    landed<0>();
    __builtin_amdgcn_s_barrier();
#define QPAM_THIN_CHUNK(J, WA, WB_, WC, H, HN)                                                  \
    load_h(HN, (J) + 1);                                                                        \
    load_w(WC, 2 * (J) + 2);                                                                    \
    landed<4 + HI>();                                                                           \
    multiply(WA, H, 2 * (J));                                                                   \
    wide::wave_lds_sync();                                                                      \
    load_w(WA, 2 * (J) + 3);                                                                    \
    landed<4 + HI>();                                                                           \
    multiply(WB_, H, 2 * (J) + 1);                                                              \
    landed<4>();                                                                                \
    __builtin_amdgcn_s_barrier();
    for (int j = 0; j < chunks; j += 6) {  // table stages repeat after 3, hidden ones after 2 chunks
        QPAM_THIN_CHUNK(j, sW0, sW1, sW2, sH0, sH1)
        if (j + 1 >= chunks) break;
        QPAM_THIN_CHUNK(j + 1, sW2, sW0, sW1, sH1, sH0)
        if (j + 2 >= chunks) break;
        QPAM_THIN_CHUNK(j + 2, sW1, sW2, sW0, sH0, sH1)
        if (j + 3 >= chunks) break;
        QPAM_THIN_CHUNK(j + 3, sW0, sW1, sW2, sH1, sH0)
        if (j + 4 >= chunks) break;
        QPAM_THIN_CHUNK(j + 4, sW2, sW0, sW1, sH0, sH1)
        if (j + 5 >= chunks) break;
        QPAM_THIN_CHUNK(j + 5, sW1, sW2, sW0, sH1, sH0)
    }
#undef QPAM_THIN_CHUNK
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // no direct load outlives the wave
    // acc[mi][r]: table row v0 + 4 g + r, hidden row 16 mi + l16
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        float m = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (v0 + 4 * g + r < a.V) m = fmaxf(m, acc[mi][r]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (token[mi] >= 0 && token[mi] == v0 + 4 * g + r) p.token_x[16 * mi + l16] = acc[mi][r];  // as keep_token
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        float s = 0.f, t = 0.f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (v0 + 4 * g + r < a.V) {
                const float d = acc[mi][r] - m, e = __builtin_amdgcn_exp2f(d * p.c);
                s += e;
                t += e * d;
            }
        s += __shfl_xor(s, 16);
        t += __shfl_xor(t, 16);
        s += __shfl_xor(s, 32);
        t += __shfl_xor(t, 32);
        if (g == 0) {
            sM[w][16 * mi + l16] = m;
            sS[w][16 * mi + l16] = s;
            sT[w][16 * mi + l16] = t * p.c;
        }
    }
    __syncthreads();
    if (tid < 16 * MI && tid < a.N) {
        float m = sM[0][tid], s = sS[0][tid], t = sT[0][tid];
        for (int v = 1; v < NW; ++v) join_scores(p.c, m, s, t, sM[v][tid], sS[v][tid], sT[v][tid]);
        const int64_t o = (int64_t)tid * p.n_vt + blockIdx.x;
        p.part_m[o] = m;
        p.part_s[o] = s;
        p.part_t[o] = t;
    }
}

template <typename T, int NW>
int launch(const FwdParams &p, hipStream_t stream) {
    const dim3 grid(p.n_vt), block(64 * NW);
    if (p.a.N <= 16)
        hipLaunchKernelGGL((scores_kernel<T, 1, NW>), grid, block, 0, stream, p);
    else if (p.a.N <= 32)
        hipLaunchKernelGGL((scores_kernel<T, 2, NW>), grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL((scores_kernel<T, 4, NW>), grid, block, 0, stream, p);
    return launch_status("thin scores_kernel");
}
int blocks(int V) { return (V + 16 * waves(V) - 1) / (16 * waves(V)); }
}  // namespace thin

int round_up(int x, int m) { return (x + m - 1) / m * m; }

template <typename T> constexpr bool is_bf() { return sizeof(T) == 2; }

// bf16 with a hidden size that is a multiple of 64 takes the 256 x 256 tiles
bool use_wide(int D) { return D % wide::WK == 0; }

// vocab tile of the forward logits kernel (128 on the fp32 and narrow bf16 paths:
// the larger partial count, used to size the workspace)
template <typename T> constexpr int vocab_tile() { return is_bf<T>() ? big::BTN : VT; }
// vocab / row padding of the backward G buffers (one value per dtype, whichever
// bf16 tile runs: 256 is a multiple of both bf16 tile widths)
template <typename T> constexpr int vocab_pad() { return is_bf<T>() ? wide::TN : VT; }
template <typename T> constexpr int row_tile() { return is_bf<T>() ? big::BTM : BM; }

template <typename T>
size_t fwd_ws(const qpam_ce_fwd_args &a) {
    const int64_t n_vt = (a.V + vocab_tile<T>() - 1) / vocab_tile<T>();
    return (size_t)a.N * n_vt * 12 + 256;
}

// Rows of one backward pass.  The reference keeps the fp32 logits and softmax of
// `chunk` rows alive (8 bytes per row and vocabulary entry); a pass here covers
// as many rows as fit those bytes: bf16 G^T alone (library GEMMs, scores) takes 2 bytes,
// bf16 G and G^T (hand-written GEMMs) 4 bytes, fp32 G and G^T 8 bytes.
int pass_rows(const qpam_ce_bwd_args &a) {
    const int64_t factor = a.dtype == QPAM_BF16 ? (blas::enabled() ? 4 : 2) : 1;
    return (int)std::min<int64_t>((int64_t)a.chunk * factor, a.N);
}

template <typename T>
size_t bwd_ws_base(const qpam_ce_bwd_args &a) {
    const int64_t Vp = round_up(a.V, vocab_pad<T>()), chunk = pass_rows(a);
    const int64_t Rp = round_up((int)chunk, row_tile<T>());
    if (is_bf<T>() && blas::enabled())  // G^T and the library GEMMs' workspace
        return (size_t)(Vp * Rp * sizeof(T)) + 4 * 256 +
               std::max((size_t)big::DH_SPLITS * chunk * a.D * sizeof(float), blas::WS_BYTES) + 256;
    const int64_t elems = (int64_t)a.D * Vp + chunk * Vp + Vp * Rp + (int64_t)a.D * Rp;
    size_t bytes = (size_t)(elems * sizeof(T)) + 4 * 256;
    // bf16: split-K partials of the hand-written dH GEMM
    if (is_bf<T>()) bytes += std::max((size_t)big::DH_SPLITS * chunk * a.D * sizeof(float), blas::WS_BYTES) + 256;
    return bytes;
}

// dw_out 1 or 2 with bf16 inputs, the library GEMMs and one pass over the rows:
// the dW GEMM writes the gradient itself (beta 0) from its fp32 sums, in bf16
// or fp32
bool dw_direct(const qpam_ce_bwd_args &a) {
    return a.dw_out != 0 && a.dtype == QPAM_BF16 && blas::enabled() && pass_rows(a) >= a.N;
}

// dw_out 1 otherwise: bf16 inputs accumulate dW in fp32 after the passes' own
// workspace (V x D, 256-byte aligned) and convert it once at the end
template <typename T>
size_t bwd_ws(const qpam_ce_bwd_args &a) {
    const size_t base = bwd_ws_base<T>(a);
    if (a.dw_out != 1 || !is_bf<T>() || dw_direct(a)) return base;
    return base + 256 + (size_t)a.V * a.D * sizeof(float);
}

__global__ void __launch_bounds__(THREADS) dw_fill_kernel(float *p, int64_t rows, int cols, int64_t ld) {
    const int64_t n = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * THREADS) {
        const int64_t r = i / cols;
        p[r * ld + (i - r * cols)] = 0.f;
    }
}

__global__ void __launch_bounds__(THREADS) dw_cast_kernel(const float *src, int64_t lds, unsigned short *dst,
                                                          int64_t ldd, int64_t rows, int cols) {
    const int64_t n = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * THREADS) {
        const int64_t r = i / cols, c = i - r * cols;
        dst[r * ldd + c] = f32_to_bf16(src[r * lds + c]);
    }
}

// scores: a FwdParams with the token scores' fields set, or NULL for the loss
template <typename T>
int run_fwd(const qpam_ce_fwd_args &a, hipStream_t stream, const FwdParams *scores = nullptr) {
    FwdParams p;
    if (scores) p = *scores;
    p.a = a;
    const bool few = scores && a.N <= thin::ROWS;
    const bool wide_tiles = is_bf<T>() && use_wide(a.D);
    const tiles::Columns cols = tiles::columns(a.N, a.V);
    const bool score_tiles = scores && is_bf<T>() && !few;
    const bool small = scores && !is_bf<T>() && !few && split::small_tiles(a.N, a.V);
    p.full_vt = cols.full;
    auto tiles_of = [&](int width) { return (a.V + width - 1) / width; };
    if (few) p.n_vt = thin::blocks(a.V);
    else if (score_tiles) p.n_vt = cols.n_vt;
    else if (small) p.n_vt = tiles_of(split::tn<2>());
    else p.n_vt = tiles_of(wide_tiles ? wide::TN : vocab_tile<T>());
    char *ws = (char *)a.workspace;
    const int64_t cnt = (int64_t)a.N * p.n_vt;
    p.part_m = (float *)ws;
    p.part_s = p.part_m + cnt;
    p.part_i = (int *)(p.part_s + cnt);
    p.part_t = (float *)p.part_i;
    p.token_x = p.part_t + cnt;
    p.red = nullptr;
    int st;
    if (few) {
        st = thin::waves(a.V) == 16 ? thin::launch<T, 16>(p, stream) : thin::launch<T, 4>(p, stream);
    } else if (scores && !is_bf<T>()) {
        if (small)
            hipLaunchKernelGGL(split::scores_tile_kernel<2>, dim3(p.n_vt, (a.N + split::tm<2>() - 1) / split::tm<2>()),
                               dim3(split::TT), 0, stream, p);
        else
            hipLaunchKernelGGL(split::scores_tile_kernel<4>, dim3(p.n_vt, (a.N + split::TM - 1) / split::TM), dim3(split::TT), 0,
                               stream, p);
        st = launch_status("split scores_tile_kernel");
    } else if (score_tiles) {
        const dim3 grid(tiles::grid(p.n_vt * ((a.N + tiles::TM - 1) / tiles::TM)));
        if (cols.narrow == 2)
            hipLaunchKernelGGL(tiles::scores_tile_kernel<2>, grid, dim3(tiles::TT), 0, stream, p);
        else
            hipLaunchKernelGGL(tiles::scores_tile_kernel<4>, grid, dim3(tiles::TT), 0, stream, p);
        st = launch_status("scores_tile_kernel");
    } else if (wide_tiles) {
        // the argmax (accuracy counts) only when requested
        const void *kern = a.correct ? (const void *)wide::fwd_tile_kernel<true> : (const void *)wide::fwd_tile_kernel<false>;
        QPAM_CHECK_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)wide::KSMEM));
        dim3 grid(big::xcd_grid(p.n_vt * ((a.N + wide::TM - 1) / wide::TM)));
        if (a.correct)
            hipLaunchKernelGGL(wide::fwd_tile_kernel<true>, grid, dim3(wide::WTHREADS), wide::KSMEM, stream, p);
        else
            hipLaunchKernelGGL(wide::fwd_tile_kernel<false>, grid, dim3(wide::WTHREADS), wide::KSMEM, stream, p);
        st = launch_status("ce fwd_tile_kernel (bf16, 256 x 256)");
    } else if (is_bf<T>()) {
        QPAM_CHECK_HIP(hipFuncSetAttribute((const void *)big::fwd_tile_kernel,
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)big::SMEM));
        dim3 grid(big::xcd_grid(p.n_vt * ((a.N + big::BTM - 1) / big::BTM)));
        hipLaunchKernelGGL(big::fwd_tile_kernel, grid, dim3(THREADS), big::SMEM, stream, p);
        st = launch_status("ce fwd_tile_kernel (bf16)");
    } else {
        const size_t smem = gemm_smem<T>();
        QPAM_CHECK_HIP(hipFuncSetAttribute((const void *)ce_fwd_tile_kernel<T>,
                                           hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        dim3 grid(p.n_vt, (a.N + BM - 1) / BM);
        hipLaunchKernelGGL(ce_fwd_tile_kernel<T>, grid, dim3(THREADS), smem, stream, p);
        st = launch_status("ce_fwd_tile_kernel");
    }
    if (st) return st;
    if (scores) {
        hipLaunchKernelGGL(scores_finalize_kernel, dim3((a.N + 3) / 4), dim3(THREADS), 0, stream, p);
        return launch_status("scores_finalize_kernel");
    }
    hipLaunchKernelGGL(ce_fwd_finalize_kernel<T>, dim3((a.N + 3) / 4), dim3(THREADS), 0, stream, p);
    st = launch_status("ce_fwd_finalize_kernel");
    if (st) return st;
    if (a.loss_sum) {
        hipLaunchKernelGGL(ce_reduce_kernel, dim3(1), dim3(1024), 0, stream, p);
        st = launch_status("ce_reduce_kernel");
    }
    return st;
}

// Ranges of K (up to `most`, at least eight steps each) for a product whose tiles leave CUs
// idle: a step takes `step_us`; the ranges' fp32 sums of `outputs` values are written and read
// again at 5 MB a us, by a launch more (4 us).
int best_ranges(int64_t most, int K, double step_us, int64_t outputs) {
    most = std::min<int64_t>(most, K / 256);
    int best = 1;
    double least = K / BK * step_us;
    for (int r = 2; r <= most; ++r) {
        const double us = (double)K / BK / r * step_us + 4 + 8e-6 / 5 * outputs * r;
        if (us < least) {
            best = r;
            least = us;
        }
    }
    return best;
}

// [M][N] = A B of tiles::gemm_kernel.  Row tiles that fill whole rounds of the 256 CUs in one
// launch; the rest, if they leave half the CUs idle, with K in ranges (as many as `part` holds
// sums of).
template <bool AT>
int scores_gemm(const unsigned short *A, int64_t lda, int M, const unsigned short *B, int64_t ldb, int b_rows, int N, int K, void *out,
                int64_t ldo, int mode, float *part, size_t part_bytes, tiles::TokenTerms terms, hipStream_t stream) {
    using U = unsigned short;
    auto launch = [&](int m0, int m, int ranges, int kper, void *to, int64_t ld, int how) {
        const int tiles = ((m + tiles::TM - 1) / tiles::TM) * ((N + tiles::TN - 1) / tiles::TN);
        const tiles::TokenTerms t = AT ? tiles::TokenTerms{terms.g + m0, terms.id + m0, 0} : tiles::TokenTerms{terms.g, terms.id, m0};
        hipLaunchKernelGGL(tiles::gemm_kernel<AT>, dim3(big::xcd_grid(tiles * ranges)), dim3(tiles::TT), 0, stream,
                           AT ? A + m0 : A + (int64_t)m0 * lda, lda, m, B, ldb, b_rows, N, K, kper, ranges, to, ld,
                           ranges > 1 ? (int64_t)m * ld : 0, how, t);
        return launch_status("tiles gemm_kernel");
    };
    auto at = [&](int m) { return static_cast<char *>(out) + (int64_t)m * ldo * (mode == tiles::OUT_BF16 ? 2 : 4); };
    const int64_t n_rt = (M + tiles::TM - 1) / tiles::TM, n_ct = (N + tiles::TN - 1) / tiles::TN;
    const int full = (int)(n_rt * n_ct / 256 * 256 / n_ct), m0 = full * tiles::TM, rest = M - m0;
    int ranges = 1;
    if (rest > 0) {
        const int64_t fit = (int64_t)(part_bytes / ((size_t)rest * N * sizeof(float)));
        ranges = best_ranges(std::min(256 / ((n_rt - full) * n_ct), fit), K, 0.95, (int64_t)rest * N);
    }
    if (ranges == 1) return launch(0, M, 1, K, out, ldo, mode);
    int st = full > 0 ? launch(0, m0, 1, K, out, ldo, mode) : QPAM_OK;
    if (st) return st;
    const int kper = round_up((K + ranges - 1) / ranges, BK), n_k = (K + kper - 1) / kper;
    if (n_k == 1) return launch(m0, rest, 1, K, at(m0), ldo, mode);
    if ((st = launch(m0, rest, n_k, kper, part, N, tiles::OUT_F32))) return st;
    const dim3 grid((unsigned)(((int64_t)rest * N / 4 + THREADS - 1) / THREADS));
    if (mode == tiles::OUT_BF16)
        hipLaunchKernelGGL(split::sum_kernel<U>, grid, dim3(THREADS), 0, stream, (const float *)part, n_k, rest, N, (U *)at(m0), ldo, 0);
    else
        hipLaunchKernelGGL(split::sum_kernel<float>, grid, dim3(THREADS), 0, stream, (const float *)part, n_k, rest, N, (float *)at(m0),
                           ldo, mode == tiles::OUT_ADD ? 1 : 0);
    return launch_status("sum_kernel");
}

// dw_write: dW written (beta 0; one pass over the rows) by the library GEMM, in
// bf16 (dw_out 1) or fp32 (dw_out 2); otherwise added into the fp32 dW
int run_bwd_bf16(const qpam_ce_bwd_args &a, hipStream_t stream, const BwdParams *scores, bool dw_write = false) {
    using U = unsigned short;
    big::GroupParams q;
    BwdParams &p = q.p;
    if (scores) p = *scores;
    p.a = a;
    p.Vp = round_up(a.V, vocab_pad<U>());
    const int chunk = pass_rows(a);
    const int Rmax = round_up(chunk, big::BTM);
    const bool wide_tiles = use_wide(a.D);
    // the G-tile kernel: 256 x 256 tiles, or 256 x 128 for hidden sizes that are not
    // a multiple of 64 (Vp and Rp are multiples of both)
    const void *gkern = wide_tiles ? (const void *)wide::grad_tile_kernel : (const void *)big::grad_tile_kernel;
    const size_t gsmem = wide_tiles ? wide::KSMEM : big::SMEM;
    auto launch_grad = [&]() {
        if (scores) {
            const tiles::Columns cols = tiles::columns(p.rows, p.Vp);
            p.full_vt = cols.full;
            auto kernel = cols.narrow == 2 ? tiles::scores_grad_kernel<2> : tiles::scores_grad_kernel<4>;
            hipLaunchKernelGGL(kernel, dim3(tiles::grid(cols.n_vt * (p.Rp / tiles::TM))), dim3(tiles::TT), 0, stream, p);
            const int st = launch_status("scores_grad_kernel");
            if (st) return st;
            hipLaunchKernelGGL(scores_token_kernel<U>, dim3((p.rows + THREADS - 1) / THREADS), dim3(THREADS), 0, stream, p);
            return launch_status("scores_token_kernel");
        }
        const int tiles = (p.Vp / (wide_tiles ? wide::TN : big::BTN)) * (p.Rp / big::BTM);
        if (wide_tiles)
            hipLaunchKernelGGL(wide::grad_tile_kernel, dim3(big::xcd_grid(tiles)), dim3(wide::WTHREADS), gsmem, stream, p);
        else
            hipLaunchKernelGGL(big::grad_tile_kernel, dim3(big::xcd_grid(tiles)), dim3(THREADS), gsmem, stream, p);
        return launch_status(wide_tiles ? "ce grad_tile_kernel (bf16, 256 x 256)" : "ce grad_tile_kernel (bf16)");
    };
    U *ws = (U *)a.workspace;
    const size_t smem = big::SMEM;
    if (scores || blas::enabled()) {
        p.wt = p.gbuf = p.ht = nullptr;
        p.gtbuf = ws;
        q.dh_part = (float *)(((uintptr_t)(ws + (int64_t)p.Vp * Rmax) + 255) & ~(uintptr_t)255);
        // G^T [Vp][Rp] from the fused grad tiles, then (the loss) two library GEMMs (column-major views):
        //   dW^T[D][V] += H^T G^T-view   (m = D, n = V, k = rows)
        //   dH^T[D][rows] = W^T G-view   (m = D, n = rows, k = V)
        p.write_g = 0;
        const size_t blas_ws = std::max((size_t)big::DH_SPLITS * chunk * a.D * sizeof(float), blas::WS_BYTES);
        QPAM_CHECK_HIP(hipFuncSetAttribute(gkern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)gsmem));
        for (int r0 = 0; r0 < a.N; r0 += chunk) {
            p.row0 = r0;
            p.rows = std::min(chunk, a.N - r0);
            p.Rp = round_up(p.rows, big::BTM);
            int st = launch_grad();
            if (st) return st;
            if (scores) {
                const U *h = (const U *)a.h + (int64_t)r0 * a.ldh, *gt = (const U *)p.gtbuf;
                const int how = !dw_write ? tiles::OUT_ADD : a.dw_out == 1 ? tiles::OUT_BF16 : tiles::OUT_F32;
                const tiles::TokenTerms terms = {p.token_g, p.token_id, 0};
                if (a.dw)
                    st = scores_gemm<false>(gt, p.Rp, a.V, h, a.ldh, p.rows, a.D, round_up(p.rows, BK), a.dw, a.lddw, how, q.dh_part,
                                            blas_ws, terms, stream);
                if (st) return st;
                if (a.dh)
                    st = scores_gemm<true>(gt, p.Rp, p.rows, (const U *)a.w, a.ldw, a.V, a.D, p.Vp, (U *)a.dh + (int64_t)r0 * a.lddh,
                                           a.lddh, tiles::OUT_BF16, q.dh_part, blas_ws, terms, stream);
                if (st) return st;
                continue;
            }
            st = blas::gemm_bf16(false, false, a.D, a.V, p.rows, (const U *)a.h + (int64_t)r0 * a.ldh, a.ldh,
                                 p.gtbuf, p.Rp, dw_write ? 0.f : 1.f, a.dw, a.lddw, !(dw_write && a.dw_out == 1),
                                 q.dh_part, blas_ws, stream);
            if (st) return st;
            st = blas::gemm_bf16(false, true, a.D, p.rows, a.V, a.w, a.ldw, p.gtbuf, p.Rp, 0.f,
                                 (U *)a.dh + (int64_t)r0 * a.lddh, a.lddh, false, q.dh_part, blas_ws, stream);
            if (st) return st;
        }
        return QPAM_OK;
    }
    p.wt = ws;
    p.gbuf = ws + (int64_t)a.D * p.Vp;
    p.gtbuf = (U *)p.gbuf + (int64_t)chunk * p.Vp;
    p.ht = (U *)p.gtbuf + (int64_t)p.Vp * Rmax;
    q.dh_part = (float *)(((uintptr_t)((U *)p.ht + (int64_t)a.D * Rmax) + 255) & ~(uintptr_t)255);
    p.write_g = 1;
    QPAM_CHECK_HIP(hipFuncSetAttribute(gkern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)gsmem));
    QPAM_CHECK_HIP(hipFuncSetAttribute((const void *)big::dw_gemm_kernel,
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    QPAM_CHECK_HIP(hipFuncSetAttribute((const void *)big::dh_gemm_kernel,
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    hipLaunchKernelGGL(transpose_kernel<U>, dim3((a.D + 63) / 64, (p.Vp + 63) / 64), dim3(THREADS), 0, stream,
                       (const U *)a.w, a.ldw, a.V, a.D, (U *)p.wt, (int64_t)p.Vp, a.D, p.Vp);
    int st = launch_status("transpose_kernel(W)");
    if (st) return st;
    q.dw_ntiles_n = (a.D + big::BTN - 1) / big::BTN;
    q.n_dw = ((a.V + big::BTM - 1) / big::BTM) * q.dw_ntiles_n;
    q.dh_ntiles_n = q.dw_ntiles_n;
    q.splits = big::DH_SPLITS;
    q.ksplit = round_up((p.Vp + q.splits - 1) / q.splits, BK);
    for (int r0 = 0; r0 < a.N; r0 += chunk) {
        p.row0 = r0;
        p.rows = std::min(chunk, a.N - r0);
        p.Rp = round_up(p.rows, big::BTM);
        hipLaunchKernelGGL(transpose_kernel<U>, dim3((a.D + 63) / 64, (p.Rp + 63) / 64), dim3(THREADS), 0, stream,
                           (const U *)a.h + (int64_t)r0 * a.ldh, a.ldh, p.rows, a.D, (U *)p.ht, (int64_t)p.Rp, a.D,
                           p.Rp);
        st = launch_status("transpose_kernel(H)");
        if (st) return st;
        st = launch_grad();
        if (st) return st;
        q.dh_ntiles_m = (p.rows + big::BTM - 1) / big::BTM;
        hipLaunchKernelGGL(big::dw_gemm_kernel, dim3(big::xcd_grid(q.n_dw)), dim3(THREADS), smem, stream, q);
        st = launch_status("ce dw_gemm_kernel (bf16)");
        if (st) return st;
        hipLaunchKernelGGL(big::dh_gemm_kernel, dim3(big::xcd_grid(q.splits * q.dh_ntiles_m * q.dh_ntiles_n)),
                           dim3(THREADS), smem, stream, q);
        st = launch_status("ce dh_gemm_kernel (bf16)");
        if (st) return st;
        hipLaunchKernelGGL(big::dh_reduce_kernel, dim3(1024), dim3(THREADS), 0, stream, q);
        st = launch_status("ce dh_reduce_kernel");
        if (st) return st;
    }
    return QPAM_OK;
}

template <typename T>
int run_bwd(const qpam_ce_bwd_args &a, hipStream_t stream, const BwdParams *scores) {
    if (is_bf<T>()) return run_bwd_bf16(a, stream, scores);
    BwdParams p;
    p.a = a;
    p.write_g = 1;
    p.Vp = round_up(a.V, VT);
    const int chunk = pass_rows(a);
    const int Rmax = round_up(chunk, BM);
    T *ws = (T *)a.workspace;
    p.wt = ws;
    p.gbuf = ws + (int64_t)a.D * p.Vp;
    p.gtbuf = (T *)p.gbuf + (int64_t)chunk * p.Vp;
    p.ht = (T *)p.gtbuf + (int64_t)p.Vp * Rmax;
    const size_t smem = gemm_smem<T>();
    QPAM_CHECK_HIP(hipFuncSetAttribute((const void *)ce_grad_tile_kernel<T>,
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    QPAM_CHECK_HIP(hipFuncSetAttribute((const void *)ce_gemm_kernel<T, false>,
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    QPAM_CHECK_HIP(hipFuncSetAttribute((const void *)ce_gemm_kernel<T, true>,
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    // W^T [D][Vp] (zero-padded vocab columns)
    hipLaunchKernelGGL(transpose_kernel<T>, dim3((a.D + 63) / 64, (p.Vp + 63) / 64), dim3(THREADS), 0, stream,
                       (const T *)a.w, a.ldw, a.V, a.D, (T *)p.wt, (int64_t)p.Vp, a.D, p.Vp);
    int st = launch_status("transpose_kernel(W)");
    if (st) return st;
    for (int r0 = 0; r0 < a.N; r0 += chunk) {
        p.row0 = r0;
        p.rows = std::min(chunk, a.N - r0);
        p.Rp = round_up(p.rows, BM);
        // H^T [D][Rp] of this chunk
        hipLaunchKernelGGL(transpose_kernel<T>, dim3((a.D + 63) / 64, (p.Rp + 63) / 64), dim3(THREADS), 0, stream,
                           (const T *)a.h + (int64_t)r0 * a.ldh, a.ldh, p.rows, a.D, (T *)p.ht, (int64_t)p.Rp, a.D,
                           p.Rp);
        st = launch_status("transpose_kernel(H)");
        if (st) return st;
        hipLaunchKernelGGL(ce_grad_tile_kernel<T>, dim3(p.Vp / VT, p.Rp / BM), dim3(THREADS), smem, stream, p);
        st = launch_status("ce_grad_tile_kernel");
        if (st) return st;
        // dH[r0 .. r0+rows] = G [rows][Vp] * (W^T [D][Vp])^T
        hipLaunchKernelGGL((ce_gemm_kernel<T, false>), dim3((a.D + BN - 1) / BN, (p.rows + BM - 1) / BM),
                           dim3(THREADS), smem, stream, (const T *)p.gbuf, (int64_t)p.Vp, p.rows, (const T *)p.wt,
                           (int64_t)p.Vp, a.D, p.Vp, (void *)((T *)a.dh + (int64_t)r0 * a.lddh), a.lddh);
        st = launch_status("ce_gemm_kernel(dH)");
        if (st) return st;
        // dW [V][D] += G^T [Vp][Rp] * (H^T [D][Rp])^T
        hipLaunchKernelGGL((ce_gemm_kernel<T, true>), dim3((a.D + BN - 1) / BN, (a.V + BM - 1) / BM),
                           dim3(THREADS), smem, stream, (const T *)p.gtbuf, (int64_t)p.Rp, a.V, (const T *)p.ht,
                           (int64_t)p.Rp, a.D, p.Rp, (void *)a.dw, a.lddw);
        st = launch_status("ce_gemm_kernel(dW)");
        if (st) return st;
    }
    return QPAM_OK;
}

int validate_common(int N, int V, int D, int dtype, const void *h, int64_t ldh, const void *w, int64_t ldw,
                    const int64_t *targets, const char *who) {
    QPAM_REQUIRE(N >= 1 && V >= 1 && D >= 1, "%s: bad sizes N=%d V=%d D=%d", who, N, V, D);
    QPAM_REQUIRE(dtype == QPAM_F32 || dtype == QPAM_BF16, "%s: dtype %d", who, dtype);
    QPAM_REQUIRE(D % BK == 0, "%s: hidden size %d must be a multiple of %d", who, D, BK);
    QPAM_REQUIRE(h && w && targets, "%s: null pointer", who);
    const int vec = dtype == QPAM_F32 ? 4 : 8;
    QPAM_REQUIRE(((uintptr_t)h % 16) == 0 && ((uintptr_t)w % 16) == 0 && ldh % vec == 0 && ldw % vec == 0 &&
                     ldh >= D && ldw >= D,
                 "%s: H and W must be 16-byte aligned with leading dims multiple of %d and >= D", who, vec);
    return QPAM_OK;
}

// Ranges of the K axis that share an [M][D] product of the token scores' fp32 backward
int k_ranges(int M, int D, int K) {
    const int64_t tiles = (int64_t)((M + split::TM - 1) / split::TM) * ((D + split::TN - 1) / split::TN);
    return best_ranges(std::min<int64_t>(256 / tiles, 16), K, 1.9, (int64_t)M * D);
}
// ... and what their partial sums take at most: 16 ranges of M rows, or 256 tiles
int64_t k_ranges_part(int64_t M, int D) { return std::min<int64_t>(16 * M * D, 256ll * split::TM * split::TN); }

// Rows of one fp32 pass of the token scores: their 4-byte G^T fits the 8 bytes a row and
// vocabulary entry that `chunk` stands for twice.
int scores_f32_rows(const qpam_ce_bwd_args &a) { return (int)std::min<int64_t>(2 * (int64_t)a.chunk, a.N); }

// G^T (the rows padded to 256) and a product's partial sums
size_t scores_f32_ws(const qpam_ce_bwd_args &a) {
    const int64_t Vp = round_up(a.V, split::TN), chunk = scores_f32_rows(a), Rp = round_up((int)chunk, split::TM);
    const int64_t part = std::max(k_ranges_part(chunk, a.D), k_ranges_part(a.V, a.D));
    return (size_t)(Vp * Rp + part) * sizeof(float) + 256;
}

// Token scores in fp32: G tiles, then dH and dW (those that are asked for), all in bf16
// parts.  dW is written by the first pass and added to by the others.
int run_scores_f32(const qpam_ce_bwd_args &a, hipStream_t stream, const BwdParams &scores) {
    BwdParams p = scores;
    p.a = a;
    p.Vp = round_up(a.V, split::TN);
    const int chunk = scores_f32_rows(a);
    float *gt = (float *)a.workspace, *part = gt + (int64_t)p.Vp * round_up(chunk, split::TM);
    p.gtbuf = gt;
    // C [M][D] (+)= A B, in ranges of K where the tiles alone leave CUs idle
    auto gemm = [&](auto kernel, const char *what, int M, const float *B, int64_t ldb, int b_rows, int K, float *C, int64_t ldc,
                    int accumulate) {
        const int ranges = k_ranges(M, a.D, K), kper = round_up((K + ranges - 1) / ranges, BK), n_k = (K + kper - 1) / kper;
        hipLaunchKernelGGL(kernel, dim3((a.D + split::TN - 1) / split::TN, (M + split::TM - 1) / split::TM, n_k), dim3(split::TT), 0,
                           stream, (const float *)gt, (int64_t)p.Rp, M, B, ldb, b_rows, a.D, K, kper, n_k > 1 ? part : C,
                           n_k > 1 ? a.D : ldc, (int64_t)M * a.D, n_k > 1 ? 0 : accumulate);
        const int st = launch_status(what);
        if (st || n_k == 1) return st;
        hipLaunchKernelGGL(split::sum_kernel<float>, dim3((unsigned)(((int64_t)M * a.D / 4 + THREADS - 1) / THREADS)), dim3(THREADS), 0, stream,
                           (const float *)part, n_k, M, a.D, C, ldc, accumulate);
        return launch_status("split sum_kernel");
    };
    int st = QPAM_OK;
    for (int r0 = 0; r0 < a.N; r0 += chunk) {
        p.row0 = r0;
        p.rows = std::min(chunk, a.N - r0);
        p.Rp = round_up(p.rows, split::TM);
        if (split::small_tiles(p.rows, p.Vp))
            hipLaunchKernelGGL(split::scores_grad_kernel<2>, dim3(p.Vp / split::tn<2>(), p.Rp / split::tm<2>()), dim3(split::TT), 0,
                               stream, p);
        else
            hipLaunchKernelGGL(split::scores_grad_kernel<4>, dim3(p.Vp / split::TN, p.Rp / split::TM), dim3(split::TT), 0, stream, p);
        if ((st = launch_status("split scores_grad_kernel"))) return st;
        hipLaunchKernelGGL(scores_token_kernel<float>, dim3((p.rows + THREADS - 1) / THREADS), dim3(THREADS), 0, stream, p);
        if ((st = launch_status("scores_token_kernel"))) return st;
        // dH [rows][D] = (G^T [Vp][Rp])^T W, dW [V][D] (+)= G^T H
        if (a.dh)
            st = gemm(split::gemm_kernel<true>, "split gemm_kernel(dH)", p.rows, (const float *)a.w, a.ldw, a.V, p.Vp,
                      (float *)a.dh + (int64_t)r0 * a.lddh, a.lddh, 0);
        if (st) return st;
        if (a.dw)
            st = gemm(split::gemm_kernel<false>, "split gemm_kernel(dW)", a.V, (const float *)a.h + (int64_t)r0 * a.ldh, a.ldh, p.rows,
                      round_up(p.rows, BK), (float *)a.dw, a.lddw, r0 > 0 ? 1 : 0);
        if (st) return st;
    }
    return QPAM_OK;
}

// The backward passes with dW as a.dw_out asks for it.
int run_backward(const qpam_ce_bwd_args &a, hipStream_t s, const BwdParams *scores) {
    if (scores && a.dtype == QPAM_F32) return run_scores_f32(a, s, *scores);
    if (a.dw_out == 0) return a.dtype == QPAM_BF16 ? run_bwd<unsigned short>(a, s, scores) : run_bwd<float>(a, s, scores);
    if (dw_direct(a) || !a.dw) return run_bwd_bf16(a, s, scores, true);
    // dW accumulated in fp32 -- dw itself when it is fp32, else the workspace's tail -- from zero
    qpam_ce_bwd_args b = a;
    b.dw_out = 0;
    float *acc = static_cast<float *>(a.dw);
    int64_t ld = a.lddw;
    const bool convert = a.dw_out == 1 && a.dtype == QPAM_BF16;
    if (convert) {
        acc = (float *)(((uintptr_t)a.workspace + bwd_ws_base<unsigned short>(b) + 255) & ~(uintptr_t)255);
        ld = a.D;
    }
    const int64_t n = (int64_t)a.V * a.D;
    const dim3 grid((unsigned)std::min<int64_t>((n + THREADS - 1) / THREADS, 65536));
    hipLaunchKernelGGL(dw_fill_kernel, grid, dim3(THREADS), 0, s, acc, (int64_t)a.V, a.D, ld);
    int st = launch_status("ce dw_fill_kernel");
    if (st) return st;
    b.dw = acc;
    b.lddw = ld;
    st = a.dtype == QPAM_BF16 ? run_bwd<unsigned short>(b, s, scores) : run_bwd<float>(b, s, scores);
    if (st || !convert) return st;
    hipLaunchKernelGGL(dw_cast_kernel, grid, dim3(THREADS), 0, s, (const float *)acc, ld, (unsigned short *)a.dw, a.lddw,
                       (int64_t)a.V, a.D);
    return launch_status("ce dw_cast_kernel");
}

// qpam_linear_logprobs_args as the loss's arguments (what they share)
qpam_ce_fwd_args fwd_args(const qpam_linear_logprobs_args &a) {
    qpam_ce_fwd_args f = {};
    f.N = a.N, f.V = a.V, f.D = a.D, f.dtype = a.dtype;
    f.h = a.h, f.ldh = a.ldh, f.w = a.w, f.ldw = a.ldw;
    f.targets = a.ids, f.ignore_index = a.ignore_index;
    f.workspace = a.workspace, f.workspace_bytes = a.workspace_bytes;
    return f;
}

qpam_ce_bwd_args bwd_args(const qpam_linear_logprobs_args &a) {
    qpam_ce_bwd_args b = {};
    b.N = a.N, b.V = a.V, b.D = a.D, b.dtype = a.dtype;
    b.h = a.h, b.ldh = a.ldh, b.w = a.w, b.ldw = a.ldw;
    b.targets = a.ids, b.ignore_index = a.ignore_index;
    b.dh = a.dh, b.lddh = a.lddh, b.dw = a.dw, b.lddw = a.lddw, b.dw_out = a.dw_out;
    b.chunk = a.chunk;
    b.workspace = a.workspace, b.workspace_bytes = a.workspace_bytes;
    return b;
}

// The bf16 token scores' workspace: the loss's, then the tokens of a pass's rows (p: their places).
size_t token_ws(const qpam_ce_bwd_args &a, BwdParams *p) {
    const size_t at = (qpam_ce_bwd_workspace_size(&a) + 255) & ~(size_t)255, rows = round_up(pass_rows(a), big::BTM);
    if (p) {
        p->token_g = reinterpret_cast<float *>(static_cast<char *>(a.workspace) + at);
        p->token_id = reinterpret_cast<int *>(p->token_g + rows);
    }
    return at + rows * (sizeof(float) + sizeof(int));
}

int validate_scores(const qpam_linear_logprobs_args &a, const char *who) {
    int st = validate_common(a.N, a.V, a.D, a.dtype, a.h, a.ldh, a.w, a.ldw, a.ids, who);
    if (st) return st;
    QPAM_REQUIRE(a.temperature >= 1e-30f && a.temperature <= 1e30f, "%s: temperature %g outside 1e-30 .. 1e30", who,
                 a.temperature);
    QPAM_REQUIRE(a.V <= (1 << 30), "%s: V=%d (at most 2^30)", who, a.V);
    QPAM_REQUIRE(a.entropy && a.stats, "%s: null entropy or stats", who);
    QPAM_REQUIRE((a.N + BM - 1) / BM <= 65535, "%s: too many rows", who);
    QPAM_REQUIRE(a.ldh < (1 << 22) && a.ldw < (1 << 22), "%s: row strides of 2^22 elements or more", who);
    return QPAM_OK;
}

}  // namespace
}  // namespace ce
}  // namespace qpam

extern "C" size_t qpam_ce_fwd_workspace_size(const qpam_ce_fwd_args *a) {
    using namespace qpam::ce;
    if (!a) return 0;
    return a->dtype == QPAM_BF16 ? fwd_ws<unsigned short>(*a) : fwd_ws<float>(*a);
}

extern "C" int qpam_ce_fwd(const qpam_ce_fwd_args *a, void *stream) {
    using namespace qpam;
    using namespace qpam::ce;
    QPAM_REQUIRE(a != nullptr, "qpam_ce_fwd: null args");
    int st = validate_common(a->N, a->V, a->D, a->dtype, a->h, a->ldh, a->w, a->ldw, a->targets, "qpam_ce_fwd");
    if (st) return st;
    QPAM_REQUIRE(a->lse && a->loss, "qpam_ce_fwd: lse and loss outputs are required");
    const size_t need = qpam_ce_fwd_workspace_size(a);
    QPAM_REQUIRE(a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace % 16) == 0,
                 "qpam_ce_fwd: workspace needs %zu bytes (got %zu)", need, a->workspace_bytes);
    QPAM_REQUIRE((a->N + BM - 1) / BM <= 65535, "qpam_ce_fwd: too many rows");
    return a->dtype == QPAM_BF16 ? run_fwd<unsigned short>(*a, (hipStream_t)stream)
                                 : run_fwd<float>(*a, (hipStream_t)stream);
}

extern "C" size_t qpam_ce_bwd_workspace_size(const qpam_ce_bwd_args *a) {
    using namespace qpam::ce;
    if (!a || a->chunk < 1) return 0;
    return a->dtype == QPAM_BF16 ? bwd_ws<unsigned short>(*a) : bwd_ws<float>(*a);
}

extern "C" int qpam_ce_bwd(const qpam_ce_bwd_args *a, void *stream) {
    using namespace qpam;
    using namespace qpam::ce;
    QPAM_REQUIRE(a != nullptr, "qpam_ce_bwd: null args");
    int st = validate_common(a->N, a->V, a->D, a->dtype, a->h, a->ldh, a->w, a->ldw, a->targets, "qpam_ce_bwd");
    if (st) return st;
    QPAM_REQUIRE(a->lse && a->grad_scale && a->dh && a->dw, "qpam_ce_bwd: null lse/grad_scale/dh/dw");
    QPAM_REQUIRE(a->chunk >= 1, "qpam_ce_bwd: chunk must be >= 1");
    QPAM_REQUIRE(a->lddh >= a->D && a->lddw >= a->D, "qpam_ce_bwd: output leading dims must be >= D");
    QPAM_REQUIRE(a->dw_out >= 0 && a->dw_out <= 2, "qpam_ce_bwd: dw_out must be 0, 1 or 2");
    const size_t need = qpam_ce_bwd_workspace_size(a);
    QPAM_REQUIRE(a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace % 16) == 0,
                 "qpam_ce_bwd: workspace needs %zu bytes (got %zu)", need, a->workspace_bytes);
    return run_backward(*a, (hipStream_t)stream, nullptr);
}

extern "C" size_t qpam_linear_logprobs_fwd_workspace_size(const qpam_linear_logprobs_args *a) {
    using namespace qpam::ce;
    if (!a || a->N < 1 || a->V < 1) return 0;
    // a row's (m, s, t) of every vocab tile, and its token's logit
    auto bytes = [&](int n_vt) { return (size_t)a->N * n_vt * 12 + (size_t)a->N * 4 + 256; };
    if (a->N <= thin::ROWS) return bytes(thin::blocks(a->V));
    if (a->dtype == QPAM_BF16) return bytes(tiles::columns(a->N, a->V).n_vt);
    if (split::small_tiles(a->N, a->V)) return bytes((a->V + split::tn<2>() - 1) / split::tn<2>());
    return bytes((a->V + split::TN - 1) / split::TN);
}

extern "C" int qpam_linear_logprobs_fwd(const qpam_linear_logprobs_args *a, void *stream) {
    using namespace qpam;
    using namespace qpam::ce;
    QPAM_REQUIRE(a != nullptr, "qpam_linear_logprobs_fwd: null args");
    int st = validate_scores(*a, "qpam_linear_logprobs_fwd");
    if (st) return st;
    QPAM_REQUIRE(a->logprobs, "qpam_linear_logprobs_fwd: null logprobs");
    const size_t need = qpam_linear_logprobs_fwd_workspace_size(a);
    QPAM_REQUIRE(a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace % 16) == 0,
                 "qpam_linear_logprobs_fwd: workspace needs %zu bytes (got %zu)", need, a->workspace_bytes);
    FwdParams p = {};
    p.c = LOG2 / a->temperature;
    p.logprobs = a->logprobs;
    p.entropy = a->entropy;
    p.stats = a->stats;
    return a->dtype == QPAM_BF16 ? run_fwd<unsigned short>(fwd_args(*a), (hipStream_t)stream, &p)
                                 : run_fwd<float>(fwd_args(*a), (hipStream_t)stream, &p);
}

extern "C" size_t qpam_linear_logprobs_bwd_workspace_size(const qpam_linear_logprobs_args *a) {
    using namespace qpam::ce;
    if (!a || a->N < 1 || a->V < 1 || a->chunk < 1) return 0;
    const qpam_ce_bwd_args b = bwd_args(*a);
    return a->dtype == QPAM_F32 ? scores_f32_ws(b) : token_ws(b, nullptr);
}

extern "C" int qpam_linear_logprobs_bwd(const qpam_linear_logprobs_args *a, void *stream) {
    using namespace qpam;
    using namespace qpam::ce;
    QPAM_REQUIRE(a != nullptr, "qpam_linear_logprobs_bwd: null args");
    int st = validate_scores(*a, "qpam_linear_logprobs_bwd");
    if (st) return st;
    QPAM_REQUIRE(a->logprobs && (a->dh || a->dw), "qpam_linear_logprobs_bwd: null logprobs, or neither dh nor dw");
    QPAM_REQUIRE(a->chunk >= 1, "qpam_linear_logprobs_bwd: chunk must be >= 1");
    QPAM_REQUIRE((!a->dh || a->lddh >= a->D) && (!a->dw || a->lddw >= a->D), "qpam_linear_logprobs_bwd: output leading dims must be >= D");
    QPAM_REQUIRE(a->dw_out == 1 || a->dw_out == 2, "qpam_linear_logprobs_bwd: dw_out must be 1 or 2");
    QPAM_REQUIRE(a->dtype == QPAM_BF16 || (a->V < (1 << 22) - 256 && scores_f32_rows(bwd_args(*a)) < (1 << 22) - 256),
                 "qpam_linear_logprobs_bwd: fp32 takes V and passes of 2 chunk rows below 2^22 - 256");
    const size_t need = qpam_linear_logprobs_bwd_workspace_size(a);
    QPAM_REQUIRE(a->workspace && a->workspace_bytes >= need && ((uintptr_t)a->workspace % 16) == 0,
                 "qpam_linear_logprobs_bwd: workspace needs %zu bytes (got %zu)", need, a->workspace_bytes);
    BwdParams p = {};
    p.inv_t = 1.f / a->temperature;
    p.c = LOG2 / a->temperature;
    p.stats = a->stats;
    p.logprobs = a->logprobs;
    p.entropy = a->entropy;
    p.g_logprobs = a->g_logprobs;
    p.g_entropy = a->g_entropy;
    if (a->dtype == QPAM_BF16) token_ws(bwd_args(*a), &p);
    return run_backward(bwd_args(*a), (hipStream_t)stream, &p);
}
