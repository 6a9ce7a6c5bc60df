// Products of rows with 4-bit weights and group scales (qpam_linear4): the decode's projections
// and logits from a quarter of the bf16 bytes.
//
//   y[i][j] = sum_k x[i][k] s[j][k / group] e[j][k]  (+ b[j])
//
// e is a 4-bit float (sign, 2 bits of exponent, 1 of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6), which the
// hardware widens to bf16 without a rounding, two at a time (v_cvt_scalef32_pk_bf16_fp4), so a weight goes
// from memory into an MFMA operand through registers alone.  A group's sum of x e is formed in fp32 by the
// matrix cores and multiplied by the scale afterwards, one fp32 multiply-add per output and group: neither
// the weight s e nor anything else is rounded to bf16 on the way.  fp32 rows are cut into three bf16 parts
// (24 bits = 3 x 8, exact), three products each.
//
// A complex weight is two neighbouring codes (re, im) and is read once: of a widened pair come the operands
// (wr, -wi) and (wi, wr) of the real and of the imaginary output, a sign and a rotation away, and both meet
// the row as it stands.  (The same product as a real matrix [wr, -wi; wi, wr] reads every weight twice.)
//
// What bounds it: few rows, the launch and one trip to memory (768 -> 768 complex, one row: 3.0 us in a graph;
// a graph's empty kernel 1.9), with a large table its bytes (50261 x 1536, one row: 10.9 us, 4.0 TB/s of 5.0).
// Some hundred rows and prompts, the vector instructions beside the MFMAs: a multiply-add for every output and
// group (one a group and MFMA lane: as long as the MFMAs themselves at group 32), the widening and turning of a
// step's codes once per 64 rows (512 x 1536 -> 50261 real, group 64: 38 % of the SIMDs' cycles MFMA, 41 % other
// vector work, LDS reads without conflicts; 2000 x 768 -> 4608 complex, group 32: 42 % and 67 %).
//
// Layout (qpam_linear4 in the header): 512-byte blocks of 16 outputs x 64 inputs in the order of the MFMA's
// B operand, so a wave reads its weights as whole consecutive 8-byte lanes.
#include <algorithm>

#include "common.h"

namespace qpam {
namespace w4 {

constexpr int TR = 16;    // outputs of a weight block
constexpr int TK = 64;    // inputs of a weight block: two MFMA steps

struct Par {
    long rows;                 // x rows of this launch
    int n, kr;                 // outputs (complex ones), real inputs of the rows that the kernel reads
    int units, tiles;          // weight blocks along the inputs, along the outputs
    int scale_step;            // weight blocks that share a scale (2 of group 128)
    const void *x; long ldx;
    const unsigned char *codes;
    const unsigned short *scales;
    const float *bias;
    void *y; long ldy;
    int planes;
    int slices;                // grid slices of 8 blocks along the outputs; behind them (times splits) those of the tail
    int whole;                 // of the slices, those of the tile kernel's whole blocks; behind them blocks of half as many outputs
    int splits, share;         // ranges of `share` weight blocks along the inputs whose sums are joined by join_kernel
    floatx4 *sums;
    int tail_n, tail_k;        // of the caller's rows x
    const void *tail; long ld_tail;
};

__device__ __forceinline__ bf16x8 frag(uintx4 v) { return __builtin_bit_cast(bf16x8, v); }

// 8 codes of a word to the MFMA's operand
__device__ __forceinline__ bf16x8 widen(unsigned w) {
    uintx4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
    return frag(r);
}

// fp32 values as sums of three bf16 values, the largest last: each what is left rounded to bf16 (to nearest: 8 + 8 + 8
// bits hold the 24 and the sum is exact).  For magnitudes below FAR; NaN stays NaN.
constexpr float FAR = 3.3e38f;   // from near 2^128 on the first rounding may overflow
__device__ __forceinline__ void split(const float (&v)[8], bf16x8 (&p)[3]) {
    uintx4 part[3];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a = v[2 * j], b = v[2 * j + 1];
#pragma unroll
        for (int h = 2; h >= 0; --h) {
            const unsigned w = pack_bf16x2(a, b);
            part[h][j] = w;
            a -= __uint_as_float(w << 16);
            b -= __uint_as_float(w & 0xffff0000u);
        }
    }
#pragma unroll
    for (int h = 0; h < 3; ++h) p[h] = frag(part[h]);
}
// The same of any value (the same parts of those below FAR, so that a row's bits do not hang on its neighbours'): the
// others by cutting bits off, infinities in the last part alone (inf - inf would make NaN of them).
__device__ __forceinline__ void split_any(const float (&v)[8], bf16x8 (&p)[3]) {
    float near[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) near[j] = fabsf(v[j]) > FAR ? 0.f : v[j];
    split(near, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (!(fabsf(v[j]) > FAR)) continue;
        const float hi = __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u);
        const float r = fabsf(v[j]) == INFINITY ? 0.f : v[j] - hi, mid = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
        p[2][j] = (__bf16)hi, p[1][j] = (__bf16)mid, p[0][j] = (__bf16)(r - mid);
    }
}

__device__ __forceinline__ void put(float *y, long at, float v) { y[at] = v; }
__device__ __forceinline__ void put(unsigned short *y, long at, float v) { y[at] = (unsigned short)pack_bf16x2(v, v); }
__device__ __forceinline__ float wide(float v) { return v; }
__device__ __forceinline__ float wide(unsigned short v) { return bf16_to_f32(v); }

// Outputs whose weights stay whole (the decay logits of a projection): a wave per row and TAIL outputs, the
// inputs over its lanes, 8 at a time where they are aligned.
constexpr int TAIL = 4;
template <typename T>
__device__ void tail_dots(const Par &p, int waves) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), groups = (p.tail_n + TAIL - 1) / TAIL;
    const long block = ((long)((int)blockIdx.z - p.slices * p.splits) * gridDim.y + blockIdx.y) * 8 + blockIdx.x, pair = block * waves + wave;
    const long row = pair / groups;
    const int t0 = (int)(pair - row * groups) * TAIL;
    if (row >= p.rows) return;
    const T *x = static_cast<const T *>(p.x) + row * p.ldx, *w[TAIL];
    float s[TAIL];
#pragma unroll
    for (int t = 0; t < TAIL; ++t) w[t] = static_cast<const T *>(p.tail) + min(t0 + t, p.tail_n - 1) * p.ld_tail, s[t] = 0.f;
    constexpr int V = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    const bool whole = !(((uintptr_t)x | (uintptr_t)w[0] | (uintptr_t)(p.ld_tail * sizeof(T))) & 15);
    for (int k = V * lane; k < p.tail_k; k += 64 * V) {   // (the same order of the sums in either form)
        if (whole && k + V <= p.tail_k) {
            const vec a = *reinterpret_cast<const vec *>(x + k);
#pragma unroll
            for (int t = 0; t < TAIL; ++t) {
                const vec b = *reinterpret_cast<const vec *>(w[t] + k);
#pragma unroll
                for (int j = 0; j < V; ++j) s[t] = fmaf(wide(a[j]), wide(b[j]), s[t]);
            }
        } else {
            for (int j = k; j < min(k + V, p.tail_k); ++j)
#pragma unroll
                for (int t = 0; t < TAIL; ++t) s[t] = fmaf(wide(x[j]), wide(w[t][j]), s[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < TAIL; ++t) {
        float v = row16_sum(s[t]);
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
        if (lane == 0 && t0 + t < p.tail_n) put(static_cast<T *>(p.y), row * p.ldy + 2 * (long)p.n + t0 + t, v);
    }
}

// Where a kernel reads rows as bf16 planes [parts][rows][ldx], 16-byte aligned, whole blocks of inputs: the
// caller's where they are that, else laid out by lay_rows_kernel (fp32 rows: their three parts).
struct Rows {
    const unsigned short *x;
    long ldx, plane;
};

template <typename T>
__global__ __launch_bounds__(256) void lay_rows_kernel(const T *x, long ldx, long rows, int kr, int kp, unsigned short *out) {
    const long per = kp / 8;
    for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < rows * per; at += (long)gridDim.x * 256) {
        const long row = at / per;
        const int k = (int)(at - row * per) * 8;
        T v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < kr ? x[row * ldx + k + j] : T(0);
        unsigned short *to = out + row * kp + k;
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uintx4 *>(to) = __builtin_bit_cast(uintx4, v);
        } else {
            bf16x8 part[3];
            split_any(v, part);
#pragma unroll
            for (int h = 0; h < 3; ++h) *reinterpret_cast<bf16x8 *>(to + (long)h * rows * kp) = part[h];
        }
    }
}

template <typename T> constexpr int parts() { return sizeof(T) == 2 ? 1 : 3; }
template <bool CPLX, int NT> constexpr int columns() { return CPLX ? 2 * NT : NT; }

// The MFMA operands of one step's codes.
template <bool CPLX, int NT>
__device__ __forceinline__ void operands(const unsigned (&w)[NT], bf16x8 (&f)[columns<CPLX, NT>()]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const bf16x8 e = widen(w[t]);
        if constexpr (CPLX) {
            uintx4 a = __builtin_bit_cast(uintx4, e), b;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                b[j] = __builtin_amdgcn_alignbit(a[j], a[j], 16);
                a[j] ^= 0x80000000u;
            }
            f[2 * t] = frag(a), f[2 * t + 1] = frag(b);
        } else {
            f[t] = e;
        }
    }
}

template <typename T>
__device__ __forceinline__ void put_pair(const Par &p, long row, int col, float re, float im) {
    T *y = static_cast<T *>(p.y) + row * p.ldy;
    if (p.bias) re += p.bias[2 * (long)col], im += p.bias[2 * (long)col + 1];
    if (p.planes) {
        put(y, col, re);
        put(y, (long)p.n + col, im);
    } else if constexpr (sizeof(T) == 2) {
        const unsigned v = pack_bf16x2(re, im);
        __builtin_memcpy(y + 2 * (long)col, &v, 4);
    } else {
        const floatx2 v = {re, im};
        __builtin_memcpy(y + 2 * (long)col, &v, 8);
    }
}

// Sums of four neighbouring rows and one output (complex: its two parts).
template <typename T, bool CPLX>
__device__ __forceinline__ void finish(const Par &p, long row, int col, floatx4 a, floatx4 b) {
    if (col >= p.n) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (row + i >= p.rows) return;
        if constexpr (CPLX) put_pair<T>(p, row + i, col, a[i], b[i]);
        else put(static_cast<T *>(p.y), (row + i) * p.ldy + col, a[i] + (p.bias ? p.bias[col] : 0.f));
    }
}

// The finished sums of 16 rows by a weight tile, to y; of a range of the inputs, to where join_kernel adds them.
template <typename T, bool CPLX>
__device__ __forceinline__ void deliver(const Par &p, int split, int tile, long m, int lane, floatx4 a, floatx4 b) {
    if (p.splits == 1) {
        finish<T, CPLX>(p, m * 16 + 4 * (lane >> 4), tile * TR + (lane & 15), a, b);
    } else {
        const long ms = (p.rows + 15) / 16;
        if (tile >= p.tiles || m >= ms) return;
        floatx4 *to = p.sums + (((long)split * p.tiles + tile) * ms + m) * (CPLX ? 128 : 64) + lane;
        to[0] = a;
        if (CPLX) to[64] = b;
    }
}

// The sums of the ranges (at most SPLITS, all read before any is added), a wave per tile and 16 rows.
constexpr int SPLITS = 4;
template <typename T, bool CPLX>
__global__ __launch_bounds__(64) void join_kernel(Par p) {
    constexpr int Z = CPLX ? 2 : 1;
    const long ms = (p.rows + 15) / 16;
    const int lane = threadIdx.x, tile = blockIdx.x;
    const floatx4 *from = p.sums + (tile * ms + blockIdx.y) * Z * 64 + lane;
    floatx4 v[SPLITS][Z];
#pragma unroll
    for (int o = 0; o < SPLITS; ++o)
#pragma unroll
        for (int z = 0; z < Z; ++z) v[o][z] = from[min(o, p.splits - 1) * p.tiles * ms * Z * 64 + z * 64];
#pragma unroll
    for (int o = 1; o < SPLITS; ++o)
#pragma unroll
        for (int z = 0; z < Z; ++z)
            if (o < p.splits) v[0][z] += v[o][z];
    finish<T, CPLX>(p, (long)blockIdx.y * 16 + 4 * (lane >> 4), tile * TR + (lane & 15), v[0][0], v[0][Z - 1]);
}

// The wave's weights: where its tiles' blocks and scales begin (the same for all lanes), and what a lane adds.
template <int NT, int GU> struct Tiles {
    const unsigned char *codes[NT];
    const unsigned short *scales[NT];
    __device__ __forceinline__ Tiles(const Par &p, int tile0) {
        const int per = GU == 2 ? 2 * p.units : p.scale_step == 1 ? p.units : (p.units + 1) / 2;
#pragma unroll
        for (int t = 0; t < NT; ++t) {   // tiles behind the last read the last one, and are not written
            const long tile = min(tile0 + t, p.tiles - 1);
            codes[t] = p.codes + tile * p.units * 512;
            scales[t] = p.scales + tile * per * TR;
        }
    }
};

// A weight block of the wave: its codes and, per output, its scales (GU groups of a block).
template <int NT, int GU> struct Block {
    uintx2 w[NT];
    unsigned s[NT];
    __device__ __forceinline__ void load(const Par &p, const Tiles<NT, GU> &from, int u, int lane) {
        const int at = GU == 2 ? 2 * u : p.scale_step == 1 ? u : u >> 1;
        // (scalar base, vector offset: left to itself the compiler adds both in vector registers at each load)
        unsigned ow = lane * 8, os = (lane & 15) * 2 * GU;
        asm("" : "+v"(ow), "+v"(os));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            w[t] = *reinterpret_cast<const uintx2 *>(from.codes[t] + (long)u * 512 + ow);
            const char *sc = reinterpret_cast<const char *>(from.scales[t] + (long)at * TR) + os;
            if constexpr (GU == 2) s[t] = *reinterpret_cast<const unsigned *>(sc);
            else s[t] = *reinterpret_cast<const unsigned short *>(sc);
        }
    }
    __device__ __forceinline__ float scale(int t, int g) const {
        return __uint_as_float(GU == 2 && g ? s[t] & 0xffff0000u : s[t] << 16);
    }
};

// One weight block times the wave's rows: MFMAs into a group's sums of 16 rows, those times the scale into acc while
// the next 16 rows' MFMAs run (two sets of sums instead of one for every row: 2000 x 768 -> 4608 complex 97 -> 67 us
// with two weight tiles a wave, whose sums alone had filled the registers).
// x(m, step, h) gives the operand of 16 rows.
template <int PARTS, bool CPLX, int MT, int NT, int GU, typename X>
__device__ __forceinline__ void multiply(const Block<NT, GU> &b, floatx4 (&acc)[MT][columns<CPLX, NT>()], X &&x) {
    constexpr int NF = columns<CPLX, NT>(), STEPS = 2 / GU;
    floatx4 sum[2][NF];
    bf16x8 f[STEPS][NF];
#pragma unroll
    for (int i = 0; i <= GU * MT; ++i) {
        const int g = i / MT, m = i % MT;
        if (i < GU * MT) {
            if (m == 0) {
#pragma unroll
                for (int st = 0; st < STEPS; ++st) {
                    unsigned w[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) w[t] = b.w[t][g * STEPS + st];
                    operands<CPLX, NT>(w, f[st]);
                }
            }
#pragma unroll
            for (int st = 0; st < STEPS; ++st)
#pragma unroll
                for (int h = 0; h < PARTS; ++h) {
                    const bf16x8 xf = x(m, g * STEPS + st, h);
#pragma unroll
                    for (int n = 0; n < NF; ++n)
                        sum[i & 1][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, f[st][n], st || h ? sum[i & 1][n] : floatx4{0, 0, 0, 0}, 0, 0, 0);
                }
        }
        if (i) {
            const int pg = (i - 1) / MT, pm = (i - 1) % MT;
#pragma unroll
            for (int n = 0; n < NF; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[pm][n][j] = fmaf(b.scale(n * NT / NF, pg), sum[(i - 1) & 1][n][j], acc[pm][n][j]);
        }
    }
}

// Grid [8][row blocks][splits * slices]: block x takes outputs 8 z + x, rows y.  The row blocks of the same weights are
// on one XCD (the first axis), one after another, so they find them in its L2.  False: a block of the tail, done.
template <typename T>
__device__ __forceinline__ bool place(const Par &p, int waves, int &ct, int &split, int &first, int &end) {
    int z = blockIdx.z;
    if (z >= p.slices * p.splits) {
        tail_dots<T>(p, waves);
        return false;
    }
    split = 0, first = 0, end = p.units;
    if (p.splits > 1) {
        split = z / p.slices, z -= split * p.slices;
        first = split * p.share, end = min(first + p.share, p.units);
    }
    ct = z * 8 + blockIdx.x;
    return true;
}

// 16 bytes at any address of the type (the hardware's global loads take them off their alignment).
template <typename V> __device__ __forceinline__ V at(const void *base, unsigned bytes) {
    V v;
    __builtin_memcpy(&v, static_cast<const char *>(base) + bytes, sizeof(V));
    return v;
}

// The rows' part of a weight block, in registers: bf16 planes, or fp32 rows cut into their parts where they are used.
// `row`: what a lane adds to the first row's start, in bytes (below 2^32).  A block that ends behind the last input kr
// is read by as many values as there are, zeros beyond (the codes there are zero, but a value of the next row may be a NaN).
template <typename XT, int PARTS> struct Part {
    uintx4 v[2][PARTS];
    __device__ __forceinline__ void load(const XT *x, unsigned row, long plane, int u, int q, int kr) {
        const int k = u * TK + 8 * q;
        if ((u + 1) * TK <= kr) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int h = 0; h < PARTS; ++h) v[ks][h] = at<uintx4>(x + h * plane, row + (k + 32 * ks) * 2u);
        } else {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int h = 0; h < PARTS; ++h) {
                    const int f = k + 32 * ks;
                    ushortx8 a = {0, 0, 0, 0, 0, 0, 0, 0};
                    if (f + 8 <= kr) {
                        a = at<ushortx8>(x + h * plane, row + f * 2u);
                    } else {
#pragma unroll
                        for (int j = 0; j < 7; ++j)
                            if (f + j < kr) a[j] = at<unsigned short>(x + h * plane, row + (f + j) * 2u);
                    }
                    v[ks][h] = __builtin_bit_cast(uintx4, a);
                }
        }
    }
    __device__ __forceinline__ bool far() const { return false; }
    template <bool ANY> __device__ __forceinline__ void get(int ks, bf16x8 (&p)[PARTS]) const {
#pragma unroll
        for (int h = 0; h < PARTS; ++h) p[h] = frag(v[ks][h]);
    }
};
template <> struct Part<float, 1> {
    floatx4 v[2][2];
    __device__ __forceinline__ void load(const float *x, unsigned row, long, int u, int q, int kr) {
        const int k = u * TK + 8 * q;
        if ((u + 1) * TK <= kr) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) v[ks][e] = at<floatx4>(x, row + (k + 32 * ks + 4 * e) * 4u);
        } else {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int f = k + 32 * ks + 4 * e;
                    floatx4 a = {0, 0, 0, 0};
                    if (f + 4 <= kr) {
                        a = at<floatx4>(x, row + f * 4u);
                    } else {
#pragma unroll
                        for (int j = 0; j < 3; ++j)
                            if (f + j < kr) a[j] = at<float>(x, row + (f + j) * 4u);
                    }
                    v[ks][e] = a;
                }
        }
    }
    // Whether any lane has a value that split does not take.
    __device__ __forceinline__ bool far() const {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 16; j += 2) m = fmaxf(fmaxf(m, fabsf(v[j / 8][j / 4 % 2][j % 4])), fabsf(v[j / 8][j / 4 % 2][j % 4 + 1]));
        return __any(m > FAR);
    }
    template <bool ANY> __device__ __forceinline__ void get(int ks, bf16x8 (&p)[3]) const {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = v[ks][j / 4][j % 4];
        if (ANY) split_any(f, p);
        else split(f, p);
    }
};

// A few rows (a decode step's): a block of 16 rows by NT x 16 outputs whose waves take the weight blocks along the
// inputs in turn, each wave's next AHEAD ones in flight while it multiplies; their sums joined through LDS in the
// waves' order.  XT: bf16 planes, or float rows as they stand.
template <typename T, typename XT, bool CPLX, int NT, int GU, int WAVES, int AHEAD>
__global__ __launch_bounds__(64 * WAVES) void step_kernel(Par p, Rows r) {
    constexpr int PARTS = parts<T>(), NF = columns<CPLX, NT>(), Z = NF / NT, XP = sizeof(XT) == 4 ? 1 : PARTS;
    __shared__ floatx4 join[WAVES * NF * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int ct, split, first, end;
    if (!place<T>(p, WAVES, ct, split, first, end) || ct * NT >= p.tiles) return;
    const int q = lane >> 4;
    const long row0 = (long)blockIdx.y * 16;
    const XT *x0 = reinterpret_cast<const XT *>(r.x) + row0 * r.ldx;
    // rows behind the last read the last one, and are not written
    const unsigned row = (unsigned)min(lane & 15, (int)min(p.rows - row0, 16L) - 1) * (unsigned)r.ldx * (unsigned)sizeof(XT);
    floatx4 acc[1][NF];
#pragma unroll
    for (int n = 0; n < NF; ++n) acc[0][n] = floatx4{0, 0, 0, 0};
    const Tiles<NT, GU> tiles(p, ct * NT);
    Block<NT, GU> b[AHEAD];
    Part<XT, XP> x[AHEAD];
    auto fetch = [&](int i, int u) {  // (behind the last block: that again, not used)
        u = min(u, p.units - 1);
        b[i].load(p, tiles, u, lane);
        x[i].load(x0, row, r.plane, u, q, p.kr);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(i, first + wave + i * WAVES);
    for (int u = first + wave; u < end; u += AHEAD * WAVES) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (u + i * WAVES >= end) break;
            bf16x8 part[PARTS];
            if (!x[i].far())
                multiply<PARTS, CPLX, 1, NT, GU>(b[i], acc, [&](int m, int ks, int h) {
                    if (h == 0) x[i].template get<false>(ks, part);
                    return part[h];
                });
            else
                multiply<PARTS, CPLX, 1, NT, GU>(b[i], acc, [&](int m, int ks, int h) {
                    if (h == 0) x[i].template get<true>(ks, part);
                    return part[h];
                });
            if (u + (i + AHEAD) * WAVES < end) fetch(i, u + (i + AHEAD) * WAVES);
        }
    }
#pragma unroll
    for (int n = 0; n < NF; ++n) join[(wave * NF + n) * 64 + lane] = acc[0][n];
    __syncthreads();
    for (int slot = threadIdx.x; slot < NT * 64; slot += 64 * WAVES) {
        const int ln = slot & 63, t = slot >> 6;
        floatx4 v[Z];
#pragma unroll
        for (int z = 0; z < Z; ++z) {
            const floatx4 *from = join + (t * Z + z) * 64 + ln;
            v[z] = from[0];
#pragma unroll
            for (int o = 1; o < WAVES; ++o) v[z] += from[o * NF * 64];
        }
        deliver<T, CPLX>(p, split, ct * NT + t, blockIdx.y, ln, v[0], v[Z - 1]);
    }
}

// More rows: WN waves side by side of MT x 16 rows by NT x 16 outputs, WK times along the inputs; the rows of the
// weight blocks at hand through LDS in the MFMA's order (direct loads, AHEAD buffers), the weights through
// registers.  A round is U weight blocks of the wave (two, where there are many: half the barriers, the LDS reads of
// the second under the products of the first: 512 x 1536 -> 50261 real 98 -> 93 us).  With WK > 1 (a decode step's
// rows, where there are few blocks) the sums are joined through LDS.
// `tile`: the block's first weight tile.
template <typename T, bool CPLX, int WN, int WK, int MT, int NT, int GU, int AHEAD, int U>
__device__ __forceinline__ void tile_block(const Par &p, const Rows &r, uintx4 *stage, int tile) {
    constexpr int PARTS = parts<T>(), NF = columns<CPLX, NT>(), Z = NF / NT, WAVES = WN * WK, PIECES = PARTS * MT * 2 * U,
                  EACH = (PIECES + WN - 1) / WN;
    // (the waves load alike, so that the loads in flight can be counted: where PIECES is no multiple of WN some twice)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wk = wave / WN;
    if (tile >= p.tiles) return;
    const int l16 = lane & 15, q = lane >> 4, tile0 = tile + wn * NT;
    const long row0 = (long)blockIdx.y * MT * 16;
    const int last = (int)min(p.rows - row0, (long)MT * 16) - 1;
    const unsigned short *x0[EACH];   // a piece's place in the first row, and what a lane adds (bytes, below 2^32)
    unsigned row[EACH];
    int block[EACH];                  // of the round's
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int piece = (i * WN + wn) % PIECES, ks = piece & 1, m = (piece >> 1) % MT, h = (piece >> 1) / MT % PARTS, un = (piece >> 1) / (MT * PARTS);
        block[i] = un;
        x0[i] = r.x + row0 * r.ldx + h * r.plane + 32 * ks;
        row[i] = ((unsigned)min(m * 16 + l16, last) * (unsigned)r.ldx + 8 * q) * 2;
    }
    const Tiles<NT, GU> tiles(p, tile0);
    Block<NT, GU> b[AHEAD][U];
    // The round from block u on into buffer i (behind the last block: that again, so that the loads in flight can be counted).
    auto fetch = [&](int i, int u) {
        uintx4 *to = stage + (i * WK + wk) * PIECES * 64;
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const unsigned *>(reinterpret_cast<const char *>(x0[j] + (long)min(u + block[j], p.units - 1) * TK) + row[j]),
                                             reinterpret_cast<unsigned *>(to + (j * WN + wn) % PIECES * 64), 16, 0, 0);
#pragma unroll
        for (int e = 0; e < U; ++e) b[i][e].load(p, tiles, min(u + e, p.units - 1), lane);
    };
    floatx4 acc[MT][NF];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[m][n] = floatx4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < AHEAD - 1; ++i) fetch(i, (wk + i * WK) * U);
    const int rounds = (p.units + WK * U - 1) / (WK * U);
    for (int v = 0; v < rounds; v += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (v + i >= rounds) break;
            // round v + i has arrived, for every wave; the buffer of the one before is free
            stage_barrier<(AHEAD - 2) * (EACH + 2 * NT * U)>();
            const int u = (wk + (v + i) * WK) * U;
            fetch((i + AHEAD - 1) % AHEAD, u + (AHEAD - 1) * WK * U);
#pragma unroll
            for (int e = 0; e < U; ++e) {
                if ((WK > 1 || e) && u + e >= p.units) break;
                const uintx4 *from = stage + (i * WK + wk) * PIECES * 64 + e * PARTS * MT * 128 + lane;
                multiply<PARTS, CPLX, MT, NT, GU>(b[i][e], acc, [&](int m, int ks, int h) { return frag(from[((h * MT + m) * 2 + ks) * 64]); });
            }
        }
    }
    if constexpr (WK == 1) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int t = 0; t < NT; ++t)
                finish<T, CPLX>(p, row0 + m * 16 + 4 * q, (tile0 + t) * TR + l16, acc[m][t * Z], acc[m][t * Z + Z - 1]);
    } else {
        stage_barrier<0>();
        floatx4 *join = reinterpret_cast<floatx4 *>(stage);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NF; ++n) join[(wave * MT * NF + m * NF + n) * 64 + lane] = acc[m][n];
        __syncthreads();
        for (int slot = threadIdx.x; slot < WN * MT * NT * 64; slot += 64 * WAVES) {
            const int ln = slot & 63, t = (slot >> 6) % NT, m = (slot >> 6) / NT % MT, w = (slot >> 6) / (NT * MT);
            floatx4 v[Z];
#pragma unroll
            for (int z = 0; z < Z; ++z) {
                const floatx4 *from = join + (w * MT * NF + m * NF + t * Z + z) * 64 + ln;
                v[z] = from[0];
#pragma unroll
                for (int o = 1; o < WK; ++o) v[z] += from[o * WN * MT * NF * 64];
            }
            finish<T, CPLX>(p, row0 + m * 16 + 4 * (ln >> 4), (tile + w * NT + t) * TR + (ln & 15), v[0], v[Z - 1]);
        }
    }
}

template <typename T, bool CPLX, int WN, int WK, int MT, int NT, int GU, int AHEAD, int OCC, int U>
__global__ __launch_bounds__(64 * WN * WK, OCC) void tile_kernel(Par p, Rows r) {
    constexpr int STAGE = AHEAD * WK * parts<T>() * MT * 128 * U, JOIN = WK > 1 ? WN * WK * MT * columns<CPLX, NT>() * 64 : 0;
    __shared__ uintx4 stage[STAGE > JOIN ? STAGE : JOIN];   // [AHEAD][WK][U][PARTS][MT][2][64]
    const int z = blockIdx.z;
    if (z >= p.slices) {
        tail_dots<T>(p, WN * WK);
    } else if (NT == 1 || z < p.whole) {
        tile_block<T, CPLX, WN, WK, MT, NT, GU, AHEAD, U>(p, r, stage, (z * 8 + blockIdx.x) * WN * NT);
    } else if constexpr (NT > 1) {
        tile_block<T, CPLX, WN, WK, MT, NT / 2, GU, AHEAD, U>(p, r, stage, p.whole * 8 * WN * NT + ((z - p.whole) * 8 + blockIdx.x) * WN * (NT / 2));
    }
}

// ---------------------------------------------------------------- launches --

// The grid of p.slices slices by blocks of `rows` rows, with the tail's dots behind them.
dim3 grid_of(const Par &p, int rows, int waves) {
    const int row_blocks = (int)((p.rows + rows - 1) / rows);
    const long per = 8L * row_blocks * waves, dots = p.rows * ((p.tail_n + TAIL - 1) / TAIL);
    return dim3(8, row_blocks, p.slices * p.splits + (int)((dots + per - 1) / per));
}

int slices_of(int tiles, int each) { return ((tiles + each - 1) / each + 7) / 8; }

template <typename T, bool CPLX>
int join_splits(const Par &p, hipStream_t stream) {
    if (int e = launch_status("qpam_linear4")) return e;
    if (p.splits == 1) return QPAM_OK;
    join_kernel<T, CPLX><<<dim3(p.tiles, (unsigned)((p.rows + 15) / 16)), dim3(64), 0, stream>>>(p);
    return launch_status("qpam_linear4");
}

template <typename T, typename XT, bool CPLX, int NT, int GU, int WAVES, int AHEAD>
int launch_step(Par p, const Rows &r, hipStream_t stream) {
    p.slices = slices_of(p.tiles, NT);
    const dim3 grid = grid_of(p, 16, WAVES);
    step_kernel<T, XT, CPLX, NT, GU, WAVES, AHEAD><<<grid, dim3(64 * WAVES), 0, stream>>>(p, r);
    return join_splits<T, CPLX>(p, stream);
}

template <typename T, bool CPLX, int WN, int WK, int MT, int NT, int GU, int AHEAD, int OCC = 1, int U = 1>
int launch_tile(Par p, const Rows &r, hipStream_t stream) {
    p.slices = p.whole = slices_of(p.tiles, WN * NT);
    if (NT > 1) {
        // the blocks behind the last whole round of 256 (a CU each) in halves, where those are one round at most
        const long slice = 8 * ((p.rows + MT * 16 - 1) / (MT * 16)), blocks = (p.tiles + WN * NT - 1) / (WN * NT) * slice / 8;
        const int whole = (int)(blocks / 256 * 256 / slice);
        const int halves = slices_of(p.tiles - whole * 8 * WN * NT, WN * NT / 2);
        if (whole && blocks % 256 && halves * slice <= 256 + slice) p.whole = whole, p.slices = whole + halves;
    }
    const dim3 grid = grid_of(p, MT * 16, WN * WK);
    tile_kernel<T, CPLX, WN, WK, MT, NT, GU, AHEAD, OCC, U><<<grid, dim3(64 * WN * WK), 0, stream>>>(p, r);
    return join_splits<T, CPLX>(p, stream);
}

int padded(int kr) { return (kr + TK - 1) / TK * TK; }

// What a call runs: a shape of blocks (run), ranges along the inputs, and the workspace.
struct Plan {
    int shape, splits, share;
    size_t lay, sums;
};

// The shape by the number of 16 x 16 pieces of the result: as long as the GPU's 256 CUs have no more than about one
// block each, a block of fewer pieces with more waves along the inputs is done earlier; then larger ones, which
// read less.  Shapes 0, 1 and 7: the step kernel of one, two and four tiles; 2 to 6: tiles in LDS (run below).
// Measured (us in a graph, 1536 real inputs, complex / real weights; in brackets the rule's):
//   bf16, group 32           0            1            7            2          3            4            5
//   1 row, 144 pieces    [3.3 / 3.0]   4.0 / 3.4    5.4 / 4.2
//   1 row, 288            3.9 / 3.5   [4.1 / 3.5]   5.5 / 4.3
//   1 row, 1152           7.2 / 6.0    7.6 / 5.8   [9.5 / 6.8]
//   16 rows, 576          7.8 / 7.5   [6.9 / 6.5]   6.5 / 5.6
//   16 rows, 1152        12.7 / 12.6   9.7 / 8.7  [10.8 / 8.2]
//   192 rows, 288         5.9 / 5.8    5.1 / 4.7    6.4 / 5.4   [5.4 / 5.1]   6.9 / 6.8    8.2 / 7.3
//   192 rows, 576         7.7 / 7.5    6.8 / 6.4    6.6 / 5.4    7.3 / 7.1   [7.0 / 6.8]   8.3 / 7.4
//   192 rows, 1728       16.2 / 14.1  11.9 / 10.5  11.1 / 7.8   12.8 / 12.0  11.2 / 10.9  [8.6 / 7.6]  20.8 / 22.3
//   512 rows, 4608         34 / 34    23.0 / 21.8  23.4 / 15.8  26.2 / 26.1  23.7 / 23.4 [17.0]/ 15.8  21.2 /[22.6]
//   512 rows, 9216                                                                       [27.8]/ 26.0  25.1 /[23.5]
//   2000 rows, 36000                                                                       99 / 84    [69 / 48]
//   fp32, group 64: the step kernel cuts the rows itself; the others read them laid out by a launch more, counted here
//                            0            1            7            5            6
//   16 rows, 144 pieces  [5.8 / 5.7]   6.3 / 5.9    8.0 / 6.5
//   16 rows, 288          9.0 / 8.7   [6.5 / 6.1]   8.3 / 6.7
//   16 rows, 1152        19.5 / 21.8  14.4 / 12.9 [15.7 / 11.7]
//   192 rows, 1728       26.2 / 28.6  17.8 / 16.1 [15.6 / 11.1] 22.7 / 26.6   26.4
//   192 rows, 2304       33.8 / 35.0  20.4 / 19.2  21.7 / 14.4 [22.9 / 26.9]  26.4
//   512 rows, 4608         58 / 61    33.7 / 32.4  35.3 / 22.4  34.9 /[31.3] [32.0]
//   512 rows, 9216                                 61.6 / 37.5  56.9 /[36.5] [47.0]
//   2000 rows, 36000                                248 / 149    186 /[112]  [162]
// The limits were set on complex weights and are the same for 1 and 16 rows; what they cost elsewhere: up to a quarter
// where a step shape is ahead (1152 pieces of a few rows, 288 and 576 of more, real bf16 ones up to some 5000), half the
// time of real fp32 products from 2048 to some 6000 pieces.  fp32 shapes 2, 3 and 4 and the step kernels of laid fp32
// rows are of rows more than 2^24 elements apart alone.
Plan plan(const qpam_linear4_args *a) {
    const int kr = a->is_complex ? 2 * a->k : a->k, units = padded(kr) / TK, tiles = (a->n + TR - 1) / TR;
    const bool f32 = a->dtype == QPAM_F32;
    // the step kernel reads rows as they stand where a lane's offset is below 2^32, the tile kernel aligned ones of bf16 in
    // whole blocks of inputs
    const bool near = a->rows == 1 || a->ldx <= (1 << 24);
    const bool whole = !f32 && near && (uintptr_t)a->x % 16 == 0 && kr % TK == 0 && (a->rows == 1 || a->ldx % 8 == 0);
    Plan l{0, 1, units, 0, 0};
    const long pieces = (a->rows + 15) / 16 * tiles;
    if (a->rows <= 16 || (f32 && near && pieces <= 2048))
        l.shape = pieces <= 256 ? 0 : pieces <= (f32 ? 512 : 1024) ? 1 : 7;
    else if (pieces > 256)  // (shape 3: 32 rows by two tiles)
        l.shape = pieces <= 512 ? 2 : (a->rows + 31) / 32 * ((tiles + 1) / 2) <= 256 ? 3 : pieces <= (f32 ? 2048 : a->is_complex ? 12288 : 4096) ? 4 : f32 && pieces > 3000 ? 6 : 5;
    const bool step = l.shape < 2 || l.shape == 7;
    if (step ? !near : !whole) l.lay = ((size_t)a->rows * padded(kr) * 2 * (f32 ? 3 : 1) + 255) / 256 * 256;
    // few pieces of long fp32 rows: more blocks by ranges of the inputs, joined in a launch of their own (16 rows x 4608
    // inputs, 48 tiles: 11.4 -> 7.4 us; bf16 7.5 -> 7.0, not worth the memory)
    if (f32 && l.shape == 0 && pieces <= 128 && units >= 48) {
        l.splits = pieces <= 64 ? 4 : 2, l.share = (units + l.splits - 1) / l.splits;
        l.sums = (size_t)l.splits * pieces * (a->is_complex ? 2048 : 1024);
    }
    return l;
}

template <typename T, bool CPLX, int GU>
int run(const Plan &l, const Par &p, const Rows &r, hipStream_t stream) {
    typedef unsigned short B;
    constexpr bool F32 = sizeof(T) == 4;
    switch (l.shape) {
    case 0:
        if constexpr (F32)
            if (!l.lay) return launch_step<T, float, CPLX, 1, GU, 8, 2>(p, r, stream);
        return launch_step<T, B, CPLX, 1, GU, 8, F32 ? 2 : 3>(p, r, stream);
    case 1:
        if constexpr (F32)
            if (!l.lay) return launch_step<T, float, CPLX, 2, GU, 8, 1>(p, r, stream);
        return launch_step<T, B, CPLX, 2, GU, 8, F32 ? 1 : 2>(p, r, stream);
    case 7:
        if constexpr (F32)
            if (!l.lay) return launch_step<T, float, CPLX, 4, GU, 8, 1>(p, r, stream);
        return launch_step<T, B, CPLX, 4, GU, 8, F32 ? 1 : 2>(p, r, stream);
    case 2: return launch_tile<T, CPLX, 2, 4, 1, 1, GU, F32 ? 2 : 3>(p, r, stream);
    case 3:
        if constexpr (F32) return launch_tile<T, CPLX, 4, 2, 1, 1, GU, 2>(p, r, stream);
        else return launch_tile<T, CPLX, 2, 4, 2, 1, GU, 3>(p, r, stream);
    case 4: return launch_tile<T, CPLX, 4, 2, 2, 1, GU, F32 ? 2 : 3>(p, r, stream);
    default:
        if constexpr (F32 && CPLX) {
            if (l.shape == 5) return launch_tile<T, CPLX, 6, 1, 2, 1, GU, 2, 1, 2>(p, r, stream);
            return launch_tile<T, CPLX, 4, 1, 2, 2, GU, 2, 3, 2>(p, r, stream);
        } else if constexpr (F32) {
            return launch_tile<T, CPLX, 8, 1, 2, 2, GU, 2, 1, 2>(p, r, stream);
        } else if constexpr (CPLX) {
            return launch_tile<T, CPLX, 4, 1, 4, 2, GU, 3, 2>(p, r, stream);
        } else {
            return launch_tile<T, CPLX, 8, 1, 4, 2, GU, 2, 1, 2>(p, r, stream);
        }
    }
}

template <typename T>
int by_group(const Plan &l, const Par &p, const Rows &r, int cplx, int group, hipStream_t stream) {
    if (cplx) return group == 32 ? run<T, true, 2>(l, p, r, stream) : run<T, true, 1>(l, p, r, stream);
    return group == 32 ? run<T, false, 2>(l, p, r, stream) : run<T, false, 1>(l, p, r, stream);
}

}  // namespace w4
}  // namespace qpam

extern "C" size_t qpam_linear4_workspace_size(const qpam_linear4_args *a) {
    if (!a) return 0;
    const int64_t k = a->is_complex ? 2 * (int64_t)a->k : a->k;
    if (a->rows < 1 || a->rows > (1L << 40) || k < 1 || k > (1 << 25) || a->n < 1 || a->n > (1 << 22)) return 0;
    const qpam::w4::Plan l = qpam::w4::plan(a);
    return l.lay + l.sums;
}

extern "C" int qpam_linear4(const qpam_linear4_args *a, void *stream) {
    using namespace qpam;
    QPAM_REQUIRE(a, "qpam_linear4: null arguments");
    QPAM_REQUIRE(a->dtype == QPAM_F32 || a->dtype == QPAM_BF16, "qpam_linear4: unknown dtype %d", a->dtype);
    QPAM_REQUIRE(a->rows >= 0 && a->rows <= (1L << 40), "qpam_linear4: %ld rows", (long)a->rows);
    QPAM_REQUIRE(a->n >= 1 && a->n <= (1 << 22) && a->k >= 1 && a->k <= (1 << 24), "qpam_linear4: sizes n = %d (1 to 2^22), k = %d (1 to 2^24)",
                 a->n, a->k);
    QPAM_REQUIRE(a->group == 32 || a->group == 64 || a->group == 128, "qpam_linear4: group %d (32, 64 or 128)", a->group);
    QPAM_REQUIRE(a->tail_n >= 0 && a->tail_n <= 4096, "qpam_linear4: tail of %d outputs", a->tail_n);
    QPAM_REQUIRE(!(a->planes || a->tail_n) || a->is_complex, "qpam_linear4: planes and tail are of complex products");
    QPAM_REQUIRE(!a->tail_n || a->planes, "qpam_linear4: a tail stands behind planes");
    if (!a->rows) return QPAM_OK;
    const int kr = a->is_complex ? 2 * a->k : a->k, wide_y = (a->is_complex ? 2 : 1) * a->n + a->tail_n;
    const int elem = a->dtype == QPAM_BF16 ? 2 : 4;
    QPAM_REQUIRE(a->x && a->codes && a->scales && a->y && (!a->tail_n || a->tail), "qpam_linear4: null pointer");
    QPAM_REQUIRE((uintptr_t)a->codes % 16 == 0 && (uintptr_t)a->scales % 4 == 0, "qpam_linear4: codes or scales not aligned");
    QPAM_REQUIRE((uintptr_t)a->x % elem == 0 && (uintptr_t)a->y % elem == 0 && (uintptr_t)a->tail % elem == 0 &&
                 (uintptr_t)a->bias % 4 == 0, "qpam_linear4: pointer not aligned to its type");
    QPAM_REQUIRE((a->ldx >= kr || a->rows == 1) && (a->ldy >= wide_y || a->rows == 1) && (!a->tail_n || a->ld_tail >= kr || a->tail_n == 1),
                 "qpam_linear4: row strides shorter than the rows");
    w4::Par p{};
    p.n = a->n, p.kr = kr;
    p.units = (kr + w4::TK - 1) / w4::TK, p.scale_step = a->group == 128 ? 2 : 1, p.tiles = (a->n + w4::TR - 1) / w4::TR;
    p.ldx = a->ldx, p.ldy = a->ldy, p.ld_tail = a->ld_tail;
    p.codes = static_cast<const unsigned char *>(a->codes), p.scales = static_cast<const unsigned short *>(a->scales);
    p.bias = a->bias, p.planes = a->planes, p.tail_n = a->tail_n, p.tail_k = kr, p.tail = a->tail;
    const w4::Plan l = w4::plan(a);
    if (l.lay + l.sums && (!a->workspace || a->workspace_bytes < l.lay + l.sums || (uintptr_t)a->workspace % 16))
        return fail(QPAM_ERR_WORKSPACE, "qpam_linear4: workspace of %zu bytes (16-byte aligned) needed", l.lay + l.sums);
    p.splits = l.splits, p.share = l.share;
    p.sums = reinterpret_cast<floatx4 *>(static_cast<char *>(a->workspace) + l.lay);
    hipStream_t st = (hipStream_t)stream;
    // a launch has fewer than 2^32 threads, a grid's second axis 2^16 blocks: rows in pieces
    const long step = std::min<long>(1 << 19, std::max<long>(16, (1L << 31) / ((p.tiles + 8L) * 1024 / 16 + 64L * a->tail_n) / 16 * 16));
    for (long at = 0; at < a->rows; at += step) {
        p.rows = std::min<long>(step, a->rows - at);
        p.x = static_cast<const char *>(a->x) + at * a->ldx * elem;
        p.y = static_cast<char *>(a->y) + at * a->ldy * elem;
        w4::Rows r{static_cast<const unsigned short *>(p.x), a->ldx, 0};
        if (l.lay) {  // each piece in turn through the same memory
            const int kp = w4::padded(kr);
            unsigned short *ws = static_cast<unsigned short *>(a->workspace);
            const long blocks = std::min<long>((p.rows * (kp / 8) + 255) / 256, 1 << 20);
            if (a->dtype == QPAM_BF16)
                w4::lay_rows_kernel<<<dim3((unsigned)blocks), dim3(256), 0, st>>>(static_cast<const unsigned short *>(p.x), a->ldx, p.rows, kr, kp, ws);
            else
                w4::lay_rows_kernel<<<dim3((unsigned)blocks), dim3(256), 0, st>>>(static_cast<const float *>(p.x), a->ldx, p.rows, kr, kp, ws);
            if (const int e = launch_status("qpam_linear4")) return e;
            r = w4::Rows{ws, kp, p.rows * kp};
            p.kr = kp;
        }
        const int e = a->dtype == QPAM_BF16 ? w4::by_group<unsigned short>(l, p, r, a->is_complex, a->group, st)
                                            : w4::by_group<float>(l, p, r, a->is_complex, a->group, st);
        if (e) return e;
    }
    return QPAM_OK;
}
