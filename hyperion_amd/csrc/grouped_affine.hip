// Grouped affine map  y_r = x_r W_e + b_e  for every row r of group e, with an optional length
// normalisation  y_r <- sqrt(dim_e) y_r / (|y_r| + 1e-10)  in the epilogue: one pre-processing or
// projection matrix per recording, domain or speaker group (a chain step of
// hyperion/transforms/cent_whiten.py:25-33, lda.py:31-34, pca.py:39-42, lnorm.py:14-17 whose parameters
// depend on the row's group).
//
// Arithmetic.  Both operands are written as sums of two fp16 numbers, x = 2^-u (x0 + 2^-11 x1) with one power of
// two per row, w = 2^-v (w0 + 2^-11 w1) with one per output column, and
//     x w ~= 2^-(u + v) (x0 w0 + 2^-11 (x0 w1 + x1 w0))
// is accumulated in fp32 by v_mfma_f32_16x16x32_f16: the dropped product is 2^-22 |x w|, and a sum over d
// coordinates has d / 32 times four roundings instead of d.  The bracket is summed over the 32 coordinates of one
// instruction and added to the rest by a fused multiply-add.  The second numbers have the range of the first: written
// without the 2^11 they end 2^-33 below a row's largest magnitude, and a whitening whose coordinates span six decades
// comes out at 1.5e-5 instead of 1e-7.  Against fp32 matrix instructions this is a third to a half of the issue time of
// the same product.
//
// A row's scale has to be known before its first value is written, and the row is read once: the scale is
// taken from the chunk of coordinates at hand, kept while later chunks stay below 2^15, and lowered otherwise, with the
// sums so far multiplied by the (exact) power of two.  The largest magnitude goes to [2^14, 2^15) where a row is one
// chunk, and to [2^8, 2^9) where it may still grow: a coordinate is held to 22 bits, or to 2^-36 of the scaled unit.
//
// fp16 rows are exact in x0 and take two products: their scale is never below one, so that no value is lost.  bf16 rows
// are exact in x0 as well unless a value lies below 2^-17 of the scaled unit; a chunk says so when it is written, and
// only then takes the third product.
//
// Measured: 127 500 fp32 rows of 24 groups, 512 -> 150, 104 us (3.3 TB/s; the copy of as much 69); 115 700 bf16 rows of
// 6 groups by an order, 512 -> 200, 106 us (2.0 TB/s); 19 200 rows of 200 groups, 200 -> 77, normalised 13.5 us; 12 rows
// of 8 groups, 512 -> 200, 9.1 us, the latency of table, row number, row and norm one after the other.  The multiply-adds
// that the scaled second numbers need are 64 of a wave's instructions per k-step of a 128-row tile beside 48 products (32
// where rows have 16 bits): the first two cases take 100 and 95 us without them, with the accuracy lost.
#include "grouped.h"

#include <type_traits>

namespace hypmi_detail {

// four coordinates of a row as floats
template <typename XT>
struct Load4;
template <>
struct Load4<float> {
    static __device__ __forceinline__ f32x4 get(const float* p) { return *reinterpret_cast<const f32x4_a4*>(p); }
};
typedef unsigned short u16x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
template <>
struct Load4<_Float16> {
    static __device__ __forceinline__ f32x4 get(const _Float16* p) {
        const u16x4_a2 r = *reinterpret_cast<const u16x4_a2*>(p);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)__builtin_bit_cast(_Float16, (unsigned short)r[e]);
        return v;
    }
};
template <>
struct Load4<__bf16> {
    static __device__ __forceinline__ f32x4 get(const __bf16* p) {
        const u16x4_a2 r = *reinterpret_cast<const u16x4_a2*>(p);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __uint_as_float((unsigned)r[e] << 16);
        return v;
    }
};

constexpr int AFFINE_RUN = 8;  // tiles dealt to an XCD at a time

// x up -> x0 + 2^-11 x1 with x0 = fp16(x up), x1 = fp16(2^11 (x up - x0)), four values and a power of two `up`:
// |x up - x0 - 2^-11 x1| <= 2^-22 |x up| + 2^-36.  An infinity becomes (inf, NaN): its products are NaN.
__device__ __forceinline__ void split_wide4(f32x4 x, float up, f16x4& x0, f16x4& x1) {
    const f32x4 t = x * up;
    x0 = __builtin_convertvector(t, f16x4);
    f32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = fmaf((float)x0[i], -2048.f, t[i] * 2048.f);
    x1 = __builtin_convertvector(r, f16x4);
}

struct AffineArgs {
    const void* x;
    int64_t ldx;
    int d_in;
    const int64_t* offsets;  // [n_groups + 1]
    const int64_t* tiles;    // [n_groups + 1] prefix of ceil(size / (16 RT))
    int n_groups;
    int64_t n_tiles;
    const int32_t* order;    // row numbers grouped, or NULL
    const uint4* w;          // fragments, see grouped_weights_kernel
    const float* col;        // [n_groups][2][16 ct]: exponent of the inverse column scale (int), bias
    const int32_t* dims;     // [n_groups] or NULL
    int ct, ks, d_out;
    float* y;
    int64_t ldy;
    int cols_y;              // columns written, see hypmi_grouped_affine
    int lnorm;
};

// RT row tiles of 16 per workgroup of eight waves, which take two column tiles of 16 each.  Coordinates are taken in
// chunks: 32 for RT = 8, 64 for RT = 4 (128 and 256 do not fit the registers of four waves per SIMD: 512 -> 200 with
// 128 rows a group 31 us with 64, 33 with 128, 79 with 256), 1024 for RT = 1, where a row is usually one chunk and
// everything it needs is requested at once.  The chunk at hand sits in
// LDS as pairs in operand order (lane l of a 16 x 32 tile: row l & 15, coordinates 8 (l >> 4) .. + 7; the row is
// XORed with 4 (l >> 4) so that the four coordinate groups of a row fall into different banks when they are written),
// the next one is on its way in registers.  Memory operations of a wave complete in order, so the weights of a whole
// chunk are requested before the vectors of the next one: no product waits for a vector that comes from HBM, and two
// workgroups share a CU, one converting while the other multiplies.
template <typename XT, int RT>
__global__ __launch_bounds__(512, RT == 1 ? 1 : 4) void grouped_affine_kernel(AffineArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int TM = 16 * RT;
    constexpr int KC = RT == 8 ? 32 : RT == 4 ? 64 : 1024;
    constexpr bool F16 = std::is_same<XT, _Float16>::value, BF16 = std::is_same<XT, __bf16>::value;
    constexpr int NP = F16 ? 1 : 2;              // parts of x
    constexpr int LPR = RT == 1 ? 32 : 8;        // lanes that load one row
    constexpr int RPT = TM * LPR / 512;          // rows per thread
    constexpr int F4 = KC / (4 * LPR);           // groups of four coordinates per thread and row
    constexpr int CW = 8, NT = 2;
    constexpr int KSC = KC / 32;                 // k-steps per chunk
    extern __shared__ __attribute__((aligned(16))) uint4 tile_mem[];  // two buffers, one where a row is one chunk
    constexpr int BUF = KSC * RT * NP * 64;
    __shared__ int exps[3][TM];  // a chunk's scales are still read while those of the next but one are written
    __shared__ int lowered[2];  // the chunk for which a scale was lowered last, by buffer
    __shared__ int second[2];   // the chunk in which an x1 was not zero last (bf16)
    __shared__ int rows[TM];
    __shared__ double norm[CW][TM];

    const int64_t t = xcd_task(blockIdx.x, g.n_tiles, AFFINE_RUN);
    if (t < 0) return;
    const int e = find_group(g.tiles, g.n_groups, t);
    const int64_t r0 = g.offsets[e] + (t - g.tiles[e]) * TM;
    const int64_t left = g.offsets[e + 1] - r0;
    const int nrows = left < TM ? (int)left : TM;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < TM) {
        const int64_t r = r0 + (tid < nrows ? tid : 0);
        rows[tid] = g.order ? g.order[r] : (int)r;
    }
    __syncthreads();

    // ---- loading side: this thread's rows and coordinates
    const int c = tid % LPR, rg = tid / LPR;
    const int chunks = (g.d_in + KC - 1) / KC;
    const int top_exp = chunks == 1 ? 15 : 9;
    int run[RPT];
    f32x4 v[RPT][F4];
#pragma unroll
    for (int i = 0; i < RPT; ++i) run[i] = 126;
    auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const XT* src = static_cast<const XT*>(g.x) + (int64_t)rows[rg + (512 / LPR) * i] * g.ldx;
#pragma unroll
            for (int f = 0; f < F4; ++f) {
                const int k = k0 + 4 * (c + LPR * f);
                f32x4 a = {0.f, 0.f, 0.f, 0.f};
                if (k + 4 <= g.d_in) {
                    a = Load4<XT>::get(src + k);
                } else if (k < g.d_in) {
                    for (int q = 0; q < g.d_in - k; ++q) a[q] = (float)src[k + q];
                }
                v[i][f] = a;
            }
        }
    };
    auto store = [&](int buf, int ch) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            float m = 0.f;
#pragma unroll
            for (int f = 0; f < F4; ++f)
#pragma unroll
                for (int q = 0; q < 4; ++q) m = fmaxf(m, fabsf(v[i][f][q]));
            m = dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(m)));
            if (LPR == 32) m = swap16_max(dpp_max<0x140>(m));
            const int ex = __builtin_amdgcn_frexp_expf(m);
            if (m > 0.f && ex + run[i] > 15 && (!F16 || run[i] > 0)) {
                run[i] = top_exp - ex;
                if (F16 && run[i] < 0) run[i] = 0;
                lowered[buf] = ch;
            }
            const float up = exp2_int(run[i]);
            const int row = rg + (512 / LPR) * i;
            if (c == 0) exps[ch % 3][row] = run[i];
            const int rt = row >> 4, r16 = row & 15;
#pragma unroll
            for (int f = 0; f < F4; ++f) {
                const int k = 4 * (c + LPR * f);  // inside the chunk
                if (F4 > 1 && ch * KC + 4 * LPR * f >= 32 * g.ks) break;
                const int s = k >> 5, kq = (k >> 3) & 3, half = (k >> 2) & 1;
                f16x4 x0, x1;
                split_wide4(v[i][f], up, x0, x1);
                if (BF16) {
                    const uint2 b = __builtin_bit_cast(uint2, x1);
                    if (b.x | b.y) second[buf] = ch;
                }
                f16x4* dst = reinterpret_cast<f16x4*>(
                                 &tile_mem[buf * BUF + ((s * RT + rt) * NP) * 64 + kq * 16 + (r16 ^ (4 * kq))]) + half;
                dst[0] = x0;
                if (NP == 2) dst[2 * 64] = x1;
            }
        }
    };

    // ---- computing side.  Column tiles go round the waves; odd workgroups start at the other end, so that the
    // waves with a tile more do not all sit on the same SIMD of a CU.
    const int r16 = lane & 15, kq = lane >> 4;
    const int wc = (t & 1) ? CW - 1 - wave : wave;
    const int xs = kq * 16 + (r16 ^ (4 * kq));
    const int ct0 = (int)blockIdx.y * (CW * NT) + wc, ct1 = ct0 + CW;
    const uint4* wp = g.w + lane;
    const int64_t w_tile = (int64_t)g.ks * 128;
    f32x4 acc[RT][NT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

    // the chunk loop of a wave with `tiles` column tiles
    auto walk = [&](auto tiles_tag) {
        constexpr int N = decltype(tiles_tag)::value;
        // k-steps of weights in registers: 2, 4 and 8 with tiles of 16 take 9.0, 9.7 and 10.3 us for the twelve rows above, 1
        // and 2 with tiles of 64 20.7 and 16.9 us for 40 rows a group of 512 -> 77, 20.6 and 20.4 for 128 of 200 -> 200
        constexpr int WS = RT == 8 ? 1 : 2;
        const uint4* w0p = wp + ((int64_t)e * g.ct + ct0) * w_tile;
        const uint4* w1p = wp + ((int64_t)e * g.ct + ct1) * w_tile;
        f16x8 w[WS][N > 0 ? N : 1][2];
        auto weights = [&](int slot, int s) {
            s = s < g.ks ? s : g.ks - 1;  // past the end: loaded, not used
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint4* p = (j ? w1p : w0p) + s * 128;
                w[slot][j][0] = __builtin_bit_cast(f16x8, p[0]);
                w[slot][j][1] = __builtin_bit_cast(f16x8, p[64]);
            }
        };
        auto step = [&](int buf, int slot, int s, bool third) {
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const uint4* xp = &tile_mem[buf * BUF + ((s * RT + i) * NP) * 64 + xs];
                const f16x8 x0 = __builtin_bit_cast(f16x8, xp[0]);
                f32x4 low[N > 0 ? N : 1];  // the products of order 2^-11
#pragma unroll
                for (int j = 0; j < N; ++j)
                    low[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[slot][j][1], x0, (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                if constexpr (NP == 2 && !BF16) {
                    const f16x8 x1 = __builtin_bit_cast(f16x8, xp[64]);
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        low[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[slot][j][0], x1, low[j], 0, 0, 0);
                }
#pragma unroll
                for (int j = 0; j < N; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[slot][j][0], x0, acc[i][j], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < N; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc[i][j][q] = fmaf(low[j][q], 0x1p-11f, acc[i][j][q]);
            }
            if (BF16 && third) {
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const f16x8 x1 = __builtin_bit_cast(f16x8, tile_mem[buf * BUF + ((s * RT + i) * NP + 1) * 64 + xs]);
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const f32x4 low = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[slot][j][0], x1,
                                                                                 (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc[i][j][q] = fmaf(low[q], 0x1p-11f, acc[i][j][q]);
                    }
                }
            }
        };
        // the k-steps of chunk `ch`
        auto multiply = [&](int buf, int ch) {
            const bool third = BF16 && __builtin_amdgcn_readfirstlane(second[buf]) == ch;
            if constexpr (KSC == WS) {
#pragma unroll
                for (int s = 0; s < KSC; ++s)
                    if (ch * KSC + s < g.ks) step(buf, s, s, third);
            } else {
                // a long chunk: the weights go round a ring of WS k-steps
                for (int s0 = 0; s0 < KSC; s0 += WS) {
                    if (ch * KSC + s0 >= g.ks) break;
#pragma unroll
                    for (int s = 0; s < WS; ++s) {
                        if (ch * KSC + s0 + s < g.ks) step(buf, s, s0 + s, third);
                        weights(s, ch * KSC + s0 + s + WS);
                    }
                }
            }
        };
        fetch(0);  // first: converting the rows waits for nothing else
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < WS; ++s) weights(s, s);
        __builtin_amdgcn_sched_barrier(0);
        store(0, 0);
        __syncthreads();
        for (int ch = 0; ch < chunks; ++ch) {
            const int buf = ch & 1;
            if (ch + 1 < chunks) fetch((ch + 1) * KC);
            __builtin_amdgcn_sched_barrier(0);
            if (N > 0) {
                if (ch > 0 && lowered[buf] == ch) {
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        const int by = exps[ch % 3][16 * i + r16] - exps[(ch + 2) % 3][16 * i + r16];
#pragma unroll
                        for (int j = 0; j < N; ++j)
#pragma unroll
                            for (int q = 0; q < 4; ++q) acc[i][j][q] = ldexpf(acc[i][j][q], by);
                    }
                }
                multiply(buf, ch);
            }
            if (ch + 1 < chunks) {
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (KSC == WS) {
#pragma unroll
                    for (int s = 0; s < KSC; ++s) weights(s, (ch + 1) * KSC + s);
                }
                store(buf ^ 1, ch + 1);
            }
            __syncthreads();
        }
    };
    if (ct1 < g.ct) walk(std::integral_constant<int, 2>());
    else if (ct0 < g.ct) walk(std::integral_constant<int, 1>());
    else walk(std::integral_constant<int, 0>());

    // ---- epilogue: lane holds columns 16 ctile + 4 kq .. + 3 of row 16 i + r16
    const int cp = 16 * g.ct;
    const float* col = g.col + (int64_t)e * 2 * cp;
    double ss[RT];  // squares of any fp32 number stay in range
#pragma unroll
    for (int i = 0; i < RT; ++i) ss[i] = 0.0;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int ctile = j ? ct1 : ct0;
        if (ctile >= g.ct) continue;
        const int4 sc = *reinterpret_cast<const int4*>(col + 16 * ctile + 4 * kq);
        const f32x4 b = *reinterpret_cast<const f32x4*>(col + cp + 16 * ctile + 4 * kq);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int cur = exps[(chunks - 1) % 3][16 * i + r16];
            // one shift by the sum of both exponents: neither scale alone may leave the range
            acc[i][j][0] = ldexpf(acc[i][j][0], sc.x - cur) + b[0];
            acc[i][j][1] = ldexpf(acc[i][j][1], sc.y - cur) + b[1];
            acc[i][j][2] = ldexpf(acc[i][j][2], sc.z - cur) + b[2];
            acc[i][j][3] = ldexpf(acc[i][j][3], sc.w - cur) + b[3];
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (g.lnorm) ss[i] = fma((double)acc[i][j][q], (double)acc[i][j][q], ss[i]);
        }
    }
    if (g.lnorm) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            ss[i] += __shfl_xor(ss[i], 16);
            ss[i] += __shfl_xor(ss[i], 32);
            if (kq == 0) norm[wc][16 * i + r16] = ss[i];
        }
        __syncthreads();
        const double top = sqrt((double)(g.dims ? g.dims[e] : g.d_out));
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            double s = 0.0;
#pragma unroll
            for (int w = 0; w < CW; ++w) s += norm[w][16 * i + r16];
            const float factor = (float)(top / (sqrt(s) + 1e-10));
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = acc[i][j] * factor;
        }
    }
    // two loops, so that whole quads are stored without conditions in between (127 500 rows of 150: 96 us, with a
    // choice at every quad 119)
    auto write = [&](auto whole_tag) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const int row = 16 * i + r16;
            if (row >= nrows) continue;
            float* out = g.y + (int64_t)rows[row] * g.ldy;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int ctile = j ? ct1 : ct0, c0 = 16 * ctile + 4 * kq;
                if constexpr (decltype(whole_tag)::value) {
                    if (ctile < g.ct && c0 < g.cols_y) *reinterpret_cast<f32x4*>(out + c0) = acc[i][j];
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (ctile < g.ct && c0 + q < g.cols_y) out[c0 + q] = acc[i][j][q];
                }
            }
        }
    };
    if ((g.cols_y & 3) == 0) write(std::true_type{});
    else write(std::false_type{});
#endif
}

// W [n_groups][d_in][d_out] -> operand fragments w[n_groups][ct][ks][part][lane] (16 bytes each: column
// 16 ct + (lane & 15), coordinates 32 ks + 8 (lane >> 4) .. + 7, zero outside W) and col[n_groups][2][16 ct]
// (exponent of the inverse scale as an int, bias).  One workgroup per (group, column tile).
__global__ __launch_bounds__(256) void grouped_weights_kernel(const float* __restrict__ W, const float* __restrict__ b,
                                                              int d_in, int d_out, int ct, int ks,
                                                              uint4* __restrict__ w, float* __restrict__ col) {
    __shared__ float top[16][17];
    const int64_t e = blockIdx.x / ct;
    const int j = (int)(blockIdx.x - e * ct);
    const int c = threadIdx.x & 15, kg = threadIdx.x >> 4;
    const int cc = 16 * j + c;
    const float* src = W + (e * d_in) * d_out + cc;
    float m = 0.f;
    if (cc < d_out)
        for (int k = kg; k < d_in; k += 16) {
            const float a = fabsf(src[(int64_t)k * d_out]);
            if (a <= 3.402823466e38f) m = fmaxf(m, a);
        }
    top[kg][c] = m;
    __syncthreads();
    m = 0.f;
    for (int i = 0; i < 16; ++i) m = fmaxf(m, top[i][c]);
    int up = m > 0.f ? 15 - __builtin_amdgcn_frexp_expf(m) : 0;
    if (kg == 0) {
        float* dst = col + e * 32 * ct;
        dst[cc] = __int_as_float(-up);
        dst[16 * ct + cc] = (b && cc < d_out) ? b[e * d_out + cc] : 0.f;
    }
    uint4* out = w + ((e * ct + j) * ks) * 128;
    for (int kb = kg; kb < 4 * ks; kb += 16) {  // blocks of eight coordinates
        f16x8 p0, p1;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int k = 8 * kb + q;
            const float x = (cc < d_out && k < d_in) ? ldexpf(src[(int64_t)k * d_out], up) : 0.f;
            p0[q] = (_Float16)x;
            p1[q] = (_Float16)((x - (float)p0[q]) * 2048.f);
        }
        uint4* dst = out + (kb >> 2) * 128 + (kb & 3) * 16 + c;
        dst[0] = __builtin_bit_cast(uint4, p0);
        dst[64] = __builtin_bit_cast(uint4, p1);
    }
}

// Length normalisation of rows of y by group where a row does not fit one workgroup of the product
// (more than 256 output columns): a wave per listed row, the rows in turn.
__global__ __launch_bounds__(256) void grouped_lnorm_kernel(float* __restrict__ y, int64_t ldy, int d_out,
                                                            const int64_t* __restrict__ offsets, int n_groups,
                                                            const int32_t* __restrict__ order,
                                                            const int32_t* __restrict__ dims, int64_t n) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < n; r += (int64_t)gridDim.x * 4) {
        double top = (double)d_out;
        if (dims) top = (double)dims[find_group(offsets, n_groups, r)];
        float* row = y + (order ? (int64_t)order[r] : r) * ldy;
        double s = 0.0;
        for (int k = lane; k < d_out; k += 64) s = fma((double)row[k], (double)row[k], s);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
        const float f = (float)(sqrt(top) / (sqrt(s) + 1e-10));
        for (int k = lane; k < d_out; k += 64) row[k] *= f;
    }
}

// Packing of projected rows by the maps of their group: g_k = (s_k + shift_t[k]) scale_t[k],
// h_k = (s_k + shift_n[k]) scale_n[k], q = (|g|^2 - |h|^2) / 2 into an enrol-side row [g, q, 1] and a test-side row
// [g, 1, q + c] (book_pack_kernel's arithmetic with maps [n_groups][4][K] and constants c[n_groups]).  A wave per
// row, the rows in turn; either side may be left out.
__global__ __launch_bounds__(256) void grouped_pack_kernel(const float* __restrict__ s, int64_t lds, int K,
                                                           const int64_t* __restrict__ offsets, int n_groups,
                                                           int64_t n, const float* __restrict__ maps,
                                                           const float* __restrict__ c, float* __restrict__ G1,
                                                           float* __restrict__ G2, int kp) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < n; r += (int64_t)gridDim.x * 4) {
        const int e = find_group(offsets, n_groups, r);
        const float* m = maps + (int64_t)e * 4 * K;
        const float* row = s + r * lds;
        float* out1 = G1 ? G1 + r * kp : nullptr;
        float* out2 = G2 ? G2 + r * kp : nullptr;
        float sum = 0.f;
        for (int k = lane; k < K; k += 64) {
            const float v = row[k];
            const float g = (v + m[k]) * m[K + k], h = (v + m[2 * K + k]) * m[3 * K + k];
            sum += (g - h) * (g + h);
            if (out1) out1[k] = g;
            if (out2) out2[k] = g;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        const float q = 0.5f * sum;
        for (int k = K + lane; k < kp; k += 64) {
            const int j = k - K;
            if (out1) out1[k] = j == 0 ? q : j == 1 ? 1.f : 0.f;
            if (out2) out2[k] = j == 0 ? 1.f : j == 1 ? q + c[e] : 0.f;
        }
    }
}

// Workgroups of four waves that take the rows in turn: 32 for each of 256 CUs at most
inline unsigned row_blocks(int64_t n) { return (unsigned)(n < 4 * 8192 ? (n + 3) / 4 : 8192); }

template <typename XT, int RT>
int launch_affine(const AffineArgs& g, hipStream_t stream) {
    const int per = 16;  // column tiles of a workgroup
    const int64_t gx = xcd_grid(g.n_tiles, AFFINE_RUN), gy = (g.ct + per - 1) / per;
    HYPMI_REQUIRE(fits_launch(gx, 512) && gy <= 65535, "grouped_affine: too many workgroups");
    constexpr int KC = RT == 8 ? 32 : RT == 4 ? 64 : 1024;
    const int lds = (g.d_in > KC ? 2 : 1) * KC * 16 * RT * (std::is_same<XT, _Float16>::value ? 2 : 4);
    if (lds > 48 * 1024)
        HYPMI_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&grouped_affine_kernel<XT, RT>),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    hipLaunchKernelGGL((grouped_affine_kernel<XT, RT>), dim3((unsigned)gx, (unsigned)gy), dim3(512), lds, stream, g);
    HYPMI_HIP(hipGetLastError());
    return HYPMI_OK;
}

template <typename XT>
int launch_affine_type(const AffineArgs& g, int tile_rows, hipStream_t stream) {
    switch (tile_rows) {
        case 16: return launch_affine<XT, 1>(g, stream);
        case 64: return launch_affine<XT, 4>(g, stream);
        default: return launch_affine<XT, 8>(g, stream);
    }
}

}  // namespace hypmi_detail

using namespace hypmi_detail;

extern "C" int64_t hypmi_grouped_weights_bytes(int n_groups, int d_in, int d_out) {
    if (n_groups < 0 || d_in <= 0 || d_out <= 0) return 0;
    return (int64_t)n_groups * ((d_out + 15) / 16) * ((d_in + 31) / 32) * 2048;
}

extern "C" int64_t hypmi_grouped_columns_bytes(int n_groups, int d_out) {
    if (n_groups < 0 || d_out <= 0) return 0;
    return (int64_t)n_groups * 2 * ((d_out + 15) / 16 * 16) * 4;
}

extern "C" int hypmi_grouped_weights(const float* W, const float* b, int n_groups, int d_in, int d_out, void* w,
                                     void* columns, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    HYPMI_REQUIRE(n_groups >= 0 && d_in > 0 && d_out > 0, "grouped_weights: bad shape");
    if (n_groups == 0) return HYPMI_OK;
    HYPMI_REQUIRE(W && w && columns, "grouped_weights: null pointer");
    HYPMI_REQUIRE(aligned16(w) && aligned16(columns), "grouped_weights: buffers must be 16-byte aligned");
    const int ct = (d_out + 15) / 16, ks = (d_in + 31) / 32;
    const int64_t blocks = (int64_t)n_groups * ct;
    HYPMI_REQUIRE(fits_launch(blocks, 256), "grouped_weights: too many groups");
    hipLaunchKernelGGL(grouped_weights_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, W, b, d_in, d_out, ct, ks,
                       static_cast<uint4*>(w), static_cast<float*>(columns));
    HYPMI_HIP(hipGetLastError());
    return HYPMI_OK;
}

extern "C" int hypmi_grouped_affine(const void* x, int x_type, int64_t ldx, int d_in, const int64_t* offsets,
                                    const int64_t* tiles, int tile_rows, int n_groups, int64_t n_rows,
                                    int64_t n_tiles, const int32_t* order, const void* w, const void* columns,
                                    const int32_t* dims, int d_out, int lnorm, float* y, int64_t ldy, int cols_y,
                                    void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    HYPMI_REQUIRE(fits_groups(n_groups) && n_rows >= 0 && n_tiles >= 0 && d_in > 0 && d_out > 0, "grouped_affine: bad shape");
    HYPMI_REQUIRE(n_rows <= 0x7fffffffLL, "grouped_affine: at most 2^31 - 1 rows");
    HYPMI_REQUIRE(x_type >= HYPMI_F32 && x_type <= HYPMI_BF16, "grouped_affine: vectors must be fp32, fp16 or bf16");
    HYPMI_REQUIRE(tile_rows == 16 || tile_rows == 64 || tile_rows == 128, "grouped_affine: tiles of 16, 64 or 128 rows");
    HYPMI_REQUIRE(ldx >= d_in && ldy >= d_out && ldy % 4 == 0, "grouped_affine: bad leading dimension");
    HYPMI_REQUIRE(cols_y >= d_out && cols_y <= (d_out + 3) / 4 * 4 && cols_y <= ldy,
                  "grouped_affine: %d columns to write (%d, or up to the next multiple of 4)", cols_y, d_out);
    if (n_tiles == 0) return HYPMI_OK;
    HYPMI_REQUIRE(x && offsets && tiles && w && columns && y, "grouped_affine: null pointer");
    HYPMI_REQUIRE(aligned16(w) && aligned16(columns) && aligned16(y), "grouped_affine: buffers must be 16-byte aligned");
    const int ct = (d_out + 15) / 16;
    const bool fused = lnorm && ct <= 16;
    AffineArgs g = {x, ldx, d_in, offsets, tiles, n_groups, n_tiles, order, static_cast<const uint4*>(w),
                    static_cast<const float*>(columns), dims, ct, (d_in + 31) / 32, d_out, y, ldy, cols_y, fused};
    int rc;
    switch (x_type) {
        case HYPMI_F32: rc = launch_affine_type<float>(g, tile_rows, stream); break;
        case HYPMI_F16: rc = launch_affine_type<_Float16>(g, tile_rows, stream); break;
        default: rc = launch_affine_type<__bf16>(g, tile_rows, stream); break;
    }
    if (rc != HYPMI_OK || !lnorm || fused) return rc;
    hipLaunchKernelGGL(grouped_lnorm_kernel, dim3(row_blocks(n_rows)), dim3(256), 0, stream, y, ldy, d_out, offsets,
                       n_groups, order, dims, n_rows);
    HYPMI_HIP(hipGetLastError());
    return HYPMI_OK;
}

extern "C" int hypmi_grouped_pack(const float* s, int64_t lds, int K, const int64_t* offsets, int n_groups, int64_t n_rows,
                                  const float* maps, const float* c, float* G1, float* G2, int kp, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    HYPMI_REQUIRE(K > 0 && kp >= K + 2 && lds >= K && fits_groups(n_groups) && n_rows >= 0, "grouped_pack: bad shape");
    HYPMI_REQUIRE(G1 || G2, "grouped_pack: no result asked for");
    if (n_rows == 0) return HYPMI_OK;
    HYPMI_REQUIRE(s && offsets && maps && c, "grouped_pack: null pointer");
    hipLaunchKernelGGL(grouped_pack_kernel, dim3(row_blocks(n_rows)), dim3(256), 0, stream, s, lds, K, offsets, n_groups,
                       n_rows, maps, c, G1, G2, kp);
    HYPMI_HIP(hipGetLastError());
    return HYPMI_OK;
}
