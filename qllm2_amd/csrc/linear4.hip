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
// A complex weight is two neighbouring codes (re, im) and is read once: with the rows (xr, -xi) and
// (xi, xr) made from a row x, the real and the imaginary output are two rows of one real product.  (The
// same product as a real matrix [wr, -wi; wi, wr] has every weight twice.)
//
// Layout (qpam_linear4 in the header): 1 KB blocks of 16 outputs x 128 inputs in the order of the MFMA's
// B operand, so a wave reads its weights as whole consecutive 16-byte lanes.
#include <algorithm>

#include "common.h"

namespace qpam {
namespace w4 {

constexpr int TR = 16;    // outputs of a weight block
constexpr int TK = 128;   // inputs of a weight block

struct Par {
    long rows;                 // x rows of this launch
    int n, kr;                 // outputs (complex ones), real inputs
    int chunks, tiles;         // weight blocks along the inputs, along the outputs
    const void *x; long ldx;
    const unsigned char *codes;
    const unsigned short *scales;
    const float *bias;
    void *y; long ldy;
    int planes;
    int row_blocks;            // blocks along the rows
    int col_blocks;            // blocks along the outputs, rounded up to the XCDs
    int vec;                   // 16-byte loads of x are aligned and whole
    int tail_n;
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

// 8 values of a row from input k on, zeros behind the last input
template <typename T> struct Eight;
template <> struct Eight<unsigned short> {
    uintx4 v;
    __device__ __forceinline__ void load(const unsigned short *row, int k, int kr, int vec) {
        v = uintx4{0, 0, 0, 0};
        if (vec) {
            if (k < kr) v = *reinterpret_cast<const uintx4 *>(row + k);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k + j < kr) v[j >> 1] |= (unsigned)row[k + j] << (16 * (j & 1));
        }
    }
    // the row (xr, -xi) of a complex row where im is 0, (xi, xr) where it is 1
    __device__ __forceinline__ void turn(int im) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = im ? (v[j] >> 16 | v[j] << 16) : v[j] ^ 0x80000000u;
    }
    static constexpr int PARTS = 1;
    __device__ __forceinline__ void split(bf16x8 (&p)[1]) const { p[0] = frag(v); }
};
template <> struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float *row, int k, int kr, int vec) {
        if (vec) {
            floatx4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
            if (k < kr) {
                a = *reinterpret_cast<const floatx4 *>(row + k);
                b = *reinterpret_cast<const floatx4 *>(row + k + 4);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = k + j < kr ? row[k + j] : 0.f;
        }
    }
    __device__ __forceinline__ void turn(int im) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const float a = v[j], b = v[j + 1];
            v[j] = im ? b : a;
            v[j + 1] = im ? a : -b;
        }
    }
    static constexpr int PARTS = 3;
    // v as a sum of three bf16 values, the largest last: each the leading 8 bits of what is left, so the
    // sum is exact.  Infinities and NaN stay in the first alone (inf - inf would make NaN of them).
    __device__ __forceinline__ void split(bf16x8 (&p)[3]) const {
        uintx4 hi, mid, lo;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            unsigned h[2], m[2], l[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float f = v[2 * j + e];
                h[e] = __float_as_uint(f) & 0xffff0000u;
                const float r = (h[e] & 0x7f800000u) == 0x7f800000u ? 0.f : f - __uint_as_float(h[e]);
                m[e] = __float_as_uint(r) & 0xffff0000u;
                l[e] = __float_as_uint(r - __uint_as_float(m[e]));
                // a NaN whose payload is in the low bits alone stays a NaN
                if (f != f) h[e] |= 0x400000u;
            }
            hi[j] = h[0] >> 16 | (h[1] & 0xffff0000u);
            mid[j] = m[0] >> 16 | (m[1] & 0xffff0000u);
            lo[j] = l[0] >> 16 | (l[1] & 0xffff0000u);
        }
        p[0] = frag(lo), p[1] = frag(mid), p[2] = frag(hi);
    }
};

__device__ __forceinline__ void put(float *y, long at, float v) { y[at] = v; }
__device__ __forceinline__ void put(unsigned short *y, long at, float v) { y[at] = (unsigned short)pack_bf16x2(v, v); }
__device__ __forceinline__ float wide(float v) { return v; }
__device__ __forceinline__ float wide(unsigned short v) { return bf16_to_f32(v); }

// Four neighbouring (virtual) rows of output col, finished sums.
template <typename T, bool CPLX>
__device__ __forceinline__ void store4(const Par &p, long vrow, int col, floatx4 v) {
    T *y = static_cast<T *>(p.y);
    if (col >= p.n) return;
    if constexpr (CPLX) {
        float br = 0.f, bi = 0.f;
        if (p.bias) br = p.bias[2 * (long)col], bi = p.bias[2 * (long)col + 1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long row = (vrow >> 1) + i;
            if (row >= p.rows) return;
            const long at = row * p.ldy;
            put(y, at + (p.planes ? col : 2 * (long)col), v[2 * i] + br);
            put(y, at + (p.planes ? (long)p.n + col : 2 * (long)col + 1), v[2 * i + 1] + bi);
        }
    } else {
        const float b = p.bias ? p.bias[col] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (vrow + i < p.rows) put(y, (vrow + i) * p.ldy + col, v[i] + b);
    }
}

// Outputs whose weights stay whole (the decay logits of a projection): a wave per row and output, the
// inputs over its lanes.
template <typename T>
__device__ void tail_dots(const Par &p, long block, int waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long pair = block * waves + wave;
    const long row = pair / p.tail_n;
    const int t = (int)(pair - row * p.tail_n);
    if (row >= p.rows) return;
    const T *x = static_cast<const T *>(p.x) + row * p.ldx, *w = static_cast<const T *>(p.tail) + t * p.ld_tail;
    float s = 0.f;
    for (int k = lane; k < p.kr; k += 64) s = fmaf(wide(x[k]), wide(w[k]), s);
    s = row16_sum(s);
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (lane == 0) put(static_cast<T *>(p.y), row * p.ldy + 2 * (long)p.n + t, s);
}

// A block: MT x 16 (virtual) rows by NT x 16 outputs, its waves the weight blocks along the inputs in
// turn, their sums joined through LDS in the waves' order.
template <typename T, bool CPLX, int MT, int NT, int G>
__global__ __launch_bounds__(1024) void rows_kernel(Par p) {
    extern __shared__ floatx4 join[];
    const int waves = blockDim.x >> 6, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long b = blockIdx.x, all = (long)p.col_blocks * p.row_blocks;
    if (b >= all) {
        tail_dots<T>(p, b - all, waves);
        return;
    }
    // the row blocks of one weight tile on one XCD, next to each other, so they find it in its L2
    const long per = 8L * p.row_blocks;
    const int ct = (int)(b / per) * 8 + (int)(b & 7), rb = (int)((b / 8) % p.row_blocks);
    if (ct * NT >= p.tiles) return;
    const int l16 = lane & 15, q = lane >> 4;
    const long vrow0 = (long)rb * MT * TR;
    const T *xr[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {  // rows behind the last read the last one, and are not written
        const long v = vrow0 + m * TR + l16, row = CPLX ? v >> 1 : v;
        xr[m] = static_cast<const T *>(p.x) + (row < p.rows ? row : p.rows - 1) * p.ldx;
    }
    floatx4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[m][t] = floatx4{0, 0, 0, 0};

    for (int c = wave; c < p.chunks; c += waves) {
        uintx4 w[NT];
        float s[NT][G];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int tile = min(ct * NT + t, p.tiles - 1);
            const long blk = (long)tile * p.chunks + c;
            w[t] = reinterpret_cast<const uintx4 *>(p.codes)[blk * 64 + lane];
#pragma unroll
            for (int g = 0; g < G; ++g) s[t][g] = bf16_to_f32(p.scales[(blk * TR + l16) * G + g]);
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            constexpr int STEPS = 4 / G;
            floatx4 sum[MT][NT];
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int t = 0; t < NT; ++t) sum[m][t] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const int ks = g * STEPS + st;
                bf16x8 wf[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) wf[t] = widen(w[t][ks]);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    Eight<T> x;
                    x.load(xr[m], c * TK + 32 * ks + 8 * q, p.kr, p.vec);
                    if (CPLX) x.turn(lane & 1);
                    bf16x8 part[Eight<T>::PARTS];
                    x.split(part);
#pragma unroll
                    for (int h = 0; h < Eight<T>::PARTS; ++h)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
                            sum[m][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(part[h], wf[t], sum[m][t], 0, 0, 0);
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][t][i] = fmaf(s[t][g], sum[m][t][i], acc[m][t][i]);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) join[(wave * MT * NT + m * NT + t) * 64 + lane] = acc[m][t];
    __syncthreads();
    for (int slot = threadIdx.x; slot < MT * NT * 64; slot += blockDim.x) {
        floatx4 v = join[slot];
        for (int o = 1; o < waves; ++o) v += join[o * MT * NT * 64 + slot];
        const int t = (slot >> 6) % NT, m = (slot >> 6) / NT, ln = slot & 63;
        store4<T, CPLX>(p, vrow0 + m * TR + 4 * (ln >> 4), (ct * NT + t) * TR + (ln & 15), v);
    }
}

// ---------------------------------------------------------------- more rows --
// From here on rows are bf16 planes [parts][rows][ldx], 16-byte aligned, whole blocks of 128 inputs: the
// caller's where they are that, else laid out by lay_rows_kernel (fp32 rows: their three parts).  Rows are
// the MFMA's rows as they stand; of a complex weight's codes come two operands, (wr, -wi) and (wi, wr),
// whose sums are the real and the imaginary outputs in the same lane.

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
        Eight<T> v;
        v.load(x + row * ldx, k, kr, 0);
        bf16x8 part[Eight<T>::PARTS];
        v.split(part);
#pragma unroll
        for (int h = 0; h < Eight<T>::PARTS; ++h)
            *reinterpret_cast<bf16x8 *>(out + ((long)h * rows + row) * kp + k) = part[h];
    }
}

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

// A weight block of the wave: its codes and, per output, its scales.
template <int NT, int G> struct Block {
    uintx4 w[NT];
    float s[NT][G];
    __device__ __forceinline__ void load(const Par &p, int tile0, int c, int lane) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const long blk = (long)min(tile0 + t, p.tiles - 1) * p.chunks + c;
            w[t] = reinterpret_cast<const uintx4 *>(p.codes)[blk * 64 + lane];
            const unsigned short *at = p.scales + (blk * TR + (lane & 15)) * G;
            if constexpr (G == 4) {
                const ushortx4 v = *reinterpret_cast<const ushortx4 *>(at);
#pragma unroll
                for (int g = 0; g < 4; ++g) s[t][g] = bf16_to_f32(v[g]);
            } else if constexpr (G == 2) {
                const unsigned v = *reinterpret_cast<const unsigned *>(at);
                s[t][0] = __uint_as_float(v << 16), s[t][1] = __uint_as_float(v & 0xffff0000u);
            } else {
                s[t][0] = bf16_to_f32(*at);
            }
        }
    }
};

// One weight block times the wave's rows: MFMAs into a group's sums, those times the scale into acc.
// x(m, step, h) gives the operand of 16 rows.
template <int PARTS, bool CPLX, int MT, int NT, int G, typename X>
__device__ __forceinline__ void multiply(const Block<NT, G> &b, floatx4 (&acc)[MT][columns<CPLX, NT>()], X &&x) {
    constexpr int NF = columns<CPLX, NT>(), STEPS = 4 / G;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        floatx4 sum[MT][NF];
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            const int ks = g * STEPS + st;
            unsigned w[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) w[t] = b.w[t][ks];
            bf16x8 f[NF];
            operands<CPLX, NT>(w, f);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < PARTS; ++h) {
                    const bf16x8 xf = x(m, ks, h);
#pragma unroll
                    for (int n = 0; n < NF; ++n)
                        sum[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, f[n], st || h ? sum[m][n] : floatx4{0, 0, 0, 0}, 0, 0, 0);
                }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NF; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][n][i] = fmaf(b.s[n * NT / NF][g], sum[m][n][i], acc[m][n][i]);
    }
}

// Block b's place: outputs ct (units of a block's), rows rb.  The row blocks of the same weights come one after
// another on one XCD, so they find them in its L2.
__device__ __forceinline__ bool place(const Par &p, long b, int &ct, int &rb) {
    const long per = 8L * p.row_blocks;
    ct = (int)(b / per) * 8 + (int)(b & 7), rb = (int)((b / 8) % p.row_blocks);
    return true;
}

// Some rows (a decode step's): a block of MT x 16 rows by NT x 16 outputs whose waves take the weight blocks
// along the inputs in turn, rows from the caches.
template <typename T, int PARTS, bool CPLX, int MT, int NT, int G>
__global__ __launch_bounds__(512) void step_kernel(Par p, Rows r) {
    constexpr int NF = columns<CPLX, NT>();
    extern __shared__ floatx4 join[];
    const int waves = blockDim.x >> 6, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long all = (long)p.col_blocks * p.row_blocks;
    if (blockIdx.x >= all) {
        tail_dots<T>(p, blockIdx.x - all, waves);
        return;
    }
    int ct, rb;
    place(p, blockIdx.x, ct, rb);
    if (ct * NT >= p.tiles) return;
    const int l16 = lane & 15, q = lane >> 4;
    const long row0 = (long)rb * MT * 16;
    const unsigned short *xr[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xr[m] = r.x + min(row0 + m * 16 + l16, p.rows - 1) * r.ldx + 8 * q;
    floatx4 acc[MT][NF];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[m][n] = floatx4{0, 0, 0, 0};
    for (int c = wave; c < p.chunks; c += waves) {
        Block<NT, G> b;
        b.load(p, ct * NT, c, lane);
        multiply<PARTS, CPLX, MT, NT, G>(b, acc, [&](int m, int ks, int h) {
            return *reinterpret_cast<const bf16x8 *>(xr[m] + h * r.plane + c * TK + 32 * ks);
        });
    }
    // the waves' sums, 16 rows at a time
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        if (m) __syncthreads();
#pragma unroll
        for (int n = 0; n < NF; ++n) join[(wave * NF + n) * 64 + lane] = acc[m][n];
        __syncthreads();
        for (int slot = threadIdx.x; slot < NT * 64; slot += blockDim.x) {
            const int t = slot >> 6, ln = slot & 63;
            floatx4 v[NF / NT];
#pragma unroll
            for (int z = 0; z < NF / NT; ++z) {
                v[z] = join[(t * (NF / NT) + z) * 64 + ln];
                for (int o = 1; o < waves; ++o) v[z] += join[(o * NF + t * (NF / NT) + z) * 64 + ln];
            }
            finish<T, CPLX>(p, row0 + m * 16 + 4 * (ln >> 4), (ct * NT + t) * 16 + (ln & 15), v[0], v[NF / NT - 1]);
        }
    }
}

// Many rows (a prompt's): WM x WN waves of MT x 16 rows by NT x 16 outputs; the rows of a weight block of 128
// inputs through LDS in the MFMA's order (direct loads, two buffers), the weights through registers.
template <typename T, int PARTS, bool CPLX, int WM, int WN, int MT, int NT, int G>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(Par p, Rows r) {
    constexpr int NF = columns<CPLX, NT>(), WAVES = WM * WN, MB = WM * MT, PIECES = PARTS * MB * 4;
    static_assert(PIECES % WAVES == 0, "the waves load alike");
    __shared__ uintx4 stage[2 * PIECES * 64];   // [2][PARTS][MB][4][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave % WM, wn = wave / WM;
    const long all = (long)p.col_blocks * p.row_blocks;
    if (blockIdx.x >= all) {
        tail_dots<T>(p, blockIdx.x - all, WAVES);
        return;
    }
    int ct, rb;
    place(p, blockIdx.x, ct, rb);
    if (ct * WN * NT >= p.tiles) return;
    const int l16 = lane & 15, q = lane >> 4, tile0 = (ct * WN + wn) * NT;
    const long row0 = (long)rb * MB * 16;
    auto fetch = [&](int c) {
        uintx4 *to = stage + (c & 1) * PIECES * 64;
#pragma unroll
        for (int i = 0; i < PIECES / WAVES; ++i) {
            const int piece = i * WAVES + wave, ks = piece & 3, m = (piece >> 2) % MB, h = (piece >> 2) / MB;
            const unsigned short *from = r.x + h * r.plane + min(row0 + m * 16 + l16, p.rows - 1) * r.ldx + c * TK + 32 * ks + 8 * q;
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const unsigned *>(from), reinterpret_cast<unsigned *>(to + piece * 64), 16, 0, 0);
        }
    };
    floatx4 acc[MT][NF];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NF; ++n) acc[m][n] = floatx4{0, 0, 0, 0};
    Block<NT, G> b, next;
    fetch(0);
    b.load(p, tile0, 0, lane);
    stage_barrier<0>();
    for (int c = 0; c < p.chunks; ++c) {
        if (c + 1 < p.chunks) {
            fetch(c + 1);
            next.load(p, tile0, c + 1, lane);
        }
        const uintx4 *from = stage + (c & 1) * PIECES * 64;
        multiply<PARTS, CPLX, MT, NT, G>(b, acc, [&](int m, int ks, int h) {
            return frag(from[((h * MB + wm * MT + m) * 4 + ks) * 64 + lane]);
        });
        b = next;
        stage_barrier<0>();
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
            finish<T, CPLX>(p, row0 + (wm * MT + m) * 16 + 4 * q, (tile0 + t) * 16 + l16, acc[m][t * (NF / NT)], acc[m][t * (NF / NT) + NF / NT - 1]);
}

// ---------------------------------------------------------------- launches --

template <typename T, bool CPLX, int MT, int NT, int G>
int launch_rows(Par p, int waves, hipStream_t stream) {
    p.col_blocks = ((p.tiles + NT - 1) / NT + 7) / 8 * 8;
    const long vrows = CPLX ? 2 * p.rows : p.rows;
    p.row_blocks = (int)((vrows + MT * TR - 1) / (MT * TR));
    if (waves > p.chunks) waves = p.chunks;
    const long tail_blocks = p.tail_n ? (p.rows * p.tail_n + waves - 1) / waves : 0;
    const long blocks = (long)p.col_blocks * p.row_blocks + tail_blocks;
    rows_kernel<T, CPLX, MT, NT, G><<<dim3((unsigned)blocks), dim3(64 * waves), (size_t)waves * MT * NT * 1024, stream>>>(p);
    return launch_status("qpam_linear4");
}

template <typename T, bool CPLX, int MT, int NT, int G>
int launch_step(Par p, const Rows &r, hipStream_t stream) {
    constexpr int PARTS = Eight<T>::PARTS, NF = columns<CPLX, NT>();
    p.col_blocks = ((p.tiles + NT - 1) / NT + 7) / 8 * 8;
    p.row_blocks = (int)((p.rows + MT * 16 - 1) / (MT * 16));
    // as few rounds over the inputs as 8 waves need, by as few waves as make that many
    const int rounds = (p.chunks + 7) / 8, waves = (p.chunks + rounds - 1) / rounds;
    const long tail_blocks = p.tail_n ? (p.rows * p.tail_n + waves - 1) / waves : 0;
    const long blocks = (long)p.col_blocks * p.row_blocks + tail_blocks;
    step_kernel<T, PARTS, CPLX, MT, NT, G><<<dim3((unsigned)blocks), dim3(64 * waves), (size_t)waves * NF * 1024, stream>>>(p, r);
    return launch_status("qpam_linear4");
}

template <typename T, bool CPLX, int WM, int WN, int MT, int NT, int G>
int launch_tile(Par p, const Rows &r, hipStream_t stream) {
    constexpr int PARTS = Eight<T>::PARTS;
    p.col_blocks = ((p.tiles + NT * WN - 1) / (NT * WN) + 7) / 8 * 8;
    p.row_blocks = (int)((p.rows + WM * MT * 16 - 1) / (WM * MT * 16));
    const long tail_blocks = p.tail_n ? (p.rows * p.tail_n + WM * WN - 1) / (WM * WN) : 0;
    const long blocks = (long)p.col_blocks * p.row_blocks + tail_blocks;
    tile_kernel<T, PARTS, CPLX, WM, WN, MT, NT, G><<<dim3((unsigned)blocks), dim3(64 * WM * WN), 0, stream>>>(p, r);
    return launch_status("qpam_linear4");
}

constexpr int few_rows(bool cplx) { return cplx ? 8 : 16; }
int padded(int kr) { return (kr + TK - 1) / TK * TK; }

// Rows that the kernels for more rows read as they stand.
bool stand(const qpam_linear4_args *a, int kr) {
    return a->dtype == QPAM_BF16 && kr % TK == 0 && (uintptr_t)a->x % 16 == 0 && a->ldx % 8 == 0;
}

size_t lay_bytes(const qpam_linear4_args *a) {
    const int kr = a->is_complex ? 2 * a->k : a->k;
    if (a->rows <= few_rows(a->is_complex) || stand(a, kr)) return 0;
    return (size_t)a->rows * padded(kr) * 2 * (a->dtype == QPAM_BF16 ? 1 : 3);
}

template <typename T, bool CPLX, int G>
int choose(const Par &p, const Rows &r, hipStream_t stream) {
    if (p.rows <= few_rows(CPLX)) return launch_rows<T, CPLX, 1, 1, G>(p, 16, stream);
    if (p.rows <= 16) return launch_step<T, CPLX, 1, 2, G>(p, r, stream);
    if (p.rows <= 32) return launch_step<T, CPLX, 2, 2, G>(p, r, stream);
    if (p.rows <= 400) return launch_step<T, CPLX, 4, 2, G>(p, r, stream);
    constexpr int WM = sizeof(T) == 2 ? 2 : 1;
    return launch_tile<T, CPLX, WM, 4 / WM, 4, CPLX ? 2 : 4, G>(p, r, stream);
}

template <typename T>
int by_group(const Par &p, const Rows &r, int cplx, int group, hipStream_t stream) {
    if (cplx) {
        if (group == 32) return choose<T, true, 4>(p, r, stream);
        if (group == 64) return choose<T, true, 2>(p, r, stream);
        return choose<T, true, 1>(p, r, stream);
    }
    if (group == 32) return choose<T, false, 4>(p, r, stream);
    if (group == 64) return choose<T, false, 2>(p, r, stream);
    return choose<T, false, 1>(p, r, stream);
}

}  // namespace w4
}  // namespace qpam

extern "C" size_t qpam_linear4_workspace_size(const qpam_linear4_args *a) {
    const int64_t k = a->is_complex ? 2 * (int64_t)a->k : a->k;
    if (a->rows < 1 || a->rows > (1L << 40) || k < 1 || k > (1 << 25)) return 0;
    return qpam::w4::lay_bytes(a);
}

extern "C" int qpam_linear4(const qpam_linear4_args *a, void *stream) {
    using namespace qpam;
    QPAM_REQUIRE(a, "qpam_linear4: null arguments");
    QPAM_REQUIRE(a->dtype == QPAM_F32 || a->dtype == QPAM_BF16, "qpam_linear4: unknown dtype %d", a->dtype);
    QPAM_REQUIRE(a->rows >= 0 && a->rows <= (1L << 40), "qpam_linear4: %ld rows", (long)a->rows);
    QPAM_REQUIRE(a->n >= 1 && a->n <= (1 << 24) && a->k >= 1 && a->k <= (1 << 24), "qpam_linear4: sizes n = %d, k = %d (1 to 2^24)",
                 a->n, a->k);
    QPAM_REQUIRE(a->group == 32 || a->group == 64 || a->group == 128, "qpam_linear4: group %d (32, 64 or 128)", a->group);
    QPAM_REQUIRE(a->tail_n >= 0 && a->tail_n <= 4096, "qpam_linear4: tail of %d outputs", a->tail_n);
    QPAM_REQUIRE(!(a->planes || a->tail_n) || a->is_complex, "qpam_linear4: planes and tail are of complex products");
    QPAM_REQUIRE(!a->tail_n || a->planes, "qpam_linear4: a tail stands behind planes");
    if (!a->rows) return QPAM_OK;
    const int kr = a->is_complex ? 2 * a->k : a->k, wide_y = (a->is_complex ? 2 : 1) * a->n + a->tail_n;
    const int elem = a->dtype == QPAM_BF16 ? 2 : 4;
    QPAM_REQUIRE(a->x && a->codes && a->scales && a->y && (!a->tail_n || a->tail), "qpam_linear4: null pointer");
    QPAM_REQUIRE((uintptr_t)a->codes % 16 == 0 && (uintptr_t)a->scales % 8 == 0, "qpam_linear4: codes or scales not aligned");
    QPAM_REQUIRE((uintptr_t)a->x % elem == 0 && (uintptr_t)a->y % elem == 0 && (uintptr_t)a->tail % elem == 0 &&
                 (uintptr_t)a->bias % 4 == 0, "qpam_linear4: pointer not aligned to its type");
    QPAM_REQUIRE((a->ldx >= kr || a->rows == 1) && (a->ldy >= wide_y || a->rows == 1) && (!a->tail_n || a->ld_tail >= kr || a->tail_n == 1),
                 "qpam_linear4: row strides shorter than the rows");
    w4::Par p{};
    p.n = a->n, p.kr = kr;
    p.chunks = (kr + w4::TK - 1) / w4::TK, p.tiles = (a->n + w4::TR - 1) / w4::TR;
    p.ldx = a->ldx, p.ldy = a->ldy, p.ld_tail = a->ld_tail;
    p.codes = static_cast<const unsigned char *>(a->codes), p.scales = static_cast<const unsigned short *>(a->scales);
    p.bias = a->bias, p.planes = a->planes, p.tail_n = a->tail_n, p.tail = a->tail;
    p.vec = kr % 8 == 0 && (uintptr_t)a->x % 16 == 0 && a->ldx * elem % 16 == 0;
    const size_t bytes = w4::lay_bytes(a);
    if (bytes && (!a->workspace || a->workspace_bytes < bytes || (uintptr_t)a->workspace % 16))
        return fail(QPAM_ERR_WORKSPACE, "qpam_linear4: workspace of %zu bytes (16-byte aligned) needed", bytes);
    hipStream_t st = (hipStream_t)stream;
    // a launch has fewer than 2^32 threads: rows in pieces
    const long per_block = (long)(p.tiles + 8) * 1024;
    const long step = std::max<long>(64, ((1L << 31) / per_block) * 8 / (1 + a->tail_n));
    for (long at = 0; at < a->rows; at += step) {
        p.rows = std::min<long>(step, a->rows - at);
        p.x = static_cast<const char *>(a->x) + at * a->ldx * elem;
        p.y = static_cast<char *>(a->y) + at * a->ldy * elem;
        w4::Rows r{static_cast<const unsigned short *>(p.x), a->ldx, 0};
        if (bytes) {  // each piece in turn through the same memory
            const int kp = w4::padded(kr);
            unsigned short *ws = static_cast<unsigned short *>(a->workspace);
            const long blocks = std::min<long>((p.rows * (kp / 8) + 255) / 256, 1 << 20);
            if (a->dtype == QPAM_BF16)
                w4::lay_rows_kernel<<<dim3((unsigned)blocks), dim3(256), 0, st>>>(static_cast<const unsigned short *>(p.x), a->ldx, p.rows, kr, kp, ws);
            else
                w4::lay_rows_kernel<<<dim3((unsigned)blocks), dim3(256), 0, st>>>(static_cast<const float *>(p.x), a->ldx, p.rows, kr, kp, ws);
            if (const int e = launch_status("qpam_linear4")) return e;
            r = w4::Rows{ws, kp, p.rows * kp};
        }
        const int e = a->dtype == QPAM_BF16 ? w4::by_group<unsigned short>(p, r, a->is_complex, a->group, st)
                                            : w4::by_group<float>(p, r, a->is_complex, a->group, st);
        if (e) return e;
    }
    return QPAM_OK;
}
