// Grouped second-order moments  C_e = sum_r w_r x_r x_r^T,  F_e = sum_r w_r x_r  over the rows r of every
// group e, in float64: the covariance of every recording of a batch (the per-recording PCA of
// hyperion/diarization/diar_ahc_plda.py:131-141, whose statistics are np.dot(x.T, x),
// hyperion/pdfs/core/normal.py:102-113) or of every domain of a training set, in one pass.
//
// What bounds it is the float64 multiply-add: on this chip the vector unit sustains 61 TFLOP/s of v_fma_f64
// and the float64 matrix instruction 35 (both measured over registers only, together no more than either), so
// the kernel is written for the vector unit.  A wave owns a 32 x 32 block of C.  Its four 16-lane rows take
// four consecutive samples; a lane holds two features of the block's row side (a) and two of its column side
// (b), and v_fmac_f64 with a row broadcast multiplies the a of lane i by every lane's b: four 8-byte loads per
// lane feed 64 multiply-adds, without shared memory.  The four partial sums (samples modulo four) are added at
// the end.  Only blocks on or above the diagonal are computed, and both halves are written from them.
//
// A group with more than `span` rows is cut into chunks; every chunk writes its block to a slot of the
// workspace and a second kernel adds the slots in chunk order, so results do not depend on scheduling.
#include "grouped.h"

namespace hypmi_detail {

struct GramArgs {
    const void* x;
    int64_t ldx;
    int d;
    const double* w;
    const int64_t* offsets;
    const int64_t* chunks;  // [n_groups + 1] prefix of max(1, ceil(size / GRAM_SPAN))
    const int64_t* slots;   // [n_groups + 1] the same for groups of several chunks, 0 for the others
    int n_groups;
    int64_t n_chunks;
    const int32_t* order;
    double* C;
    double* F;
    double* part;           // [slots][pairs][32 * 32], then [slots][32 nb]
    double* part_f;
    int nb, pairs;
};

constexpr int GRAM_SPAN = 1024;  // rows of one chunk

// acc[i] += a(lane i of this lane's row of 16) * b, i = 0 .. 15.  The leading s_nop covers the two wait states
// between a vector write of `a` and its use through DPP.
__device__ __forceinline__ void fma_row16(double (&acc)[16], double a, double b) {
    asm("s_nop 1\n\t"
        "v_fmac_f64_dpp %0, %16, %17 row_newbcast:0 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %1, %16, %17 row_newbcast:1 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %2, %16, %17 row_newbcast:2 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %3, %16, %17 row_newbcast:3 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %4, %16, %17 row_newbcast:4 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %5, %16, %17 row_newbcast:5 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %6, %16, %17 row_newbcast:6 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %7, %16, %17 row_newbcast:7 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %8, %16, %17 row_newbcast:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %9, %16, %17 row_newbcast:9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %10, %16, %17 row_newbcast:10 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %11, %16, %17 row_newbcast:11 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %12, %16, %17 row_newbcast:12 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %13, %16, %17 row_newbcast:13 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %14, %16, %17 row_newbcast:14 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f64_dpp %15, %16, %17 row_newbcast:15 row_mask:0xf bank_mask:0xf"
        : "+&v"(acc[0]), "+&v"(acc[1]), "+&v"(acc[2]), "+&v"(acc[3]), "+&v"(acc[4]), "+&v"(acc[5]), "+&v"(acc[6]),
          "+&v"(acc[7]), "+&v"(acc[8]), "+&v"(acc[9]), "+&v"(acc[10]), "+&v"(acc[11]), "+&v"(acc[12]), "+&v"(acc[13]),
          "+&v"(acc[14]), "+&v"(acc[15])
        : "v"(a), "v"(b));
}

// block pair p (row-major over bi <= bj) -> bi, bj
__device__ __forceinline__ void pair_of(int p, int nb, int& bi, int& bj) {
    bi = 0;
    while (p >= nb - bi) {
        p -= nb - bi;
        ++bi;
    }
    bj = bi + p;
}

template <typename XT>
__global__ __launch_bounds__(256) void grouped_gram_kernel(GramArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int quads = (g.pairs + 3) >> 2;
    const int64_t t = xcd_slot(blockIdx.x, g.n_chunks * quads);
    if (t < 0) return;
    const int64_t chunk = t / quads;
    const int pair = (int)(t - chunk * quads) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (pair >= g.pairs) return;
    const int e = find_group(g.chunks, g.n_groups, chunk);
    const int64_t ch = chunk - g.chunks[e];
    const int64_t s_beg = g.offsets[e] + ch * GRAM_SPAN;
    const int64_t s_lim = g.offsets[e + 1];
    const int ns = s_lim - s_beg < GRAM_SPAN ? (int)(s_lim - s_beg) : GRAM_SPAN;
    int bi, bj;
    pair_of(pair, g.nb, bi, bj);
    const int lane = threadIdx.x & 63, l15 = lane & 15, l4 = lane >> 4;
    const XT* X = static_cast<const XT*>(g.x);
    int fa[2], fb[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        fa[h] = 32 * bi + 16 * h + l15;
        fb[h] = 32 * bj + 16 * h + l15;
        fa[h] = fa[h] < g.d ? fa[h] : g.d - 1;
        fb[h] = fb[h] < g.d ? fb[h] : g.d - 1;
    }
    double acc[2][2][16];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.0;
    double f[2] = {0.0, 0.0};

    XT a[2], b[2];
    double ws;
    auto fetch = [&](int s) {
        const int64_t r = s_beg + (s + l4 < ns ? s + l4 : ns - 1);
        const int64_t row = g.order ? (int64_t)g.order[r] : r;
        const XT* p = X + row * g.ldx;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            a[h] = p[fa[h]];
            b[h] = p[fb[h]];
        }
        ws = s + l4 < ns ? (g.w ? g.w[row] : 1.0) : 0.0;
    };
    if (ns > 0) {
        fetch(0);
        for (int s = 0; s < ns; s += 4) {
            const bool in = s + l4 < ns;  // a row past the end is a copy of the last one: taken out by value
            double da[2], db[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                da[h] = in ? (double)a[h] : 0.0;
                db[h] = in ? (g.w ? (double)b[h] * ws : (double)b[h]) : 0.0;
            }
            if (s + 4 < ns) fetch(s + 4);
#pragma unroll
            for (int h = 0; h < 2; ++h) f[h] += db[h];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) fma_row16(acc[i][j], da[i], db[j]);
        }
    }
    // the four samples of a step
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        f[h] += __shfl_xor(f[h], 16);
        f[h] += __shfl_xor(f[h], 32);
    }
    const int64_t slot = g.slots[e + 1] > g.slots[e] ? g.slots[e] + ch : -1;
    double* part = g.part + (slot * g.pairs + pair) * 1024;
    double* C = g.C + (int64_t)e * g.d * g.d;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) {
                double v = acc[i][j][q];
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                // C[32 bi + 16 i + q][32 bj + 16 j + l15]
                if (l4 != (q & 3)) continue;  // all four rows hold the sum; they share the stores
                if (slot >= 0) {
                    part[(16 * i + q) * 32 + 16 * j + l15] = v;
                } else {
                    const int r = 32 * bi + 16 * i + q, c = 32 * bj + 16 * j + l15;
                    if (r <= c && c < g.d) {
                        C[(int64_t)r * g.d + c] = v;
                        if (r < c) C[(int64_t)c * g.d + r] = v;
                    }
                }
            }
    if (bi == bj && l4 < 2) {
        const int c = 32 * bi + 16 * l4 + l15;
        const double v = l4 ? f[1] : f[0];
        if (slot >= 0) g.part_f[slot * 32 * g.nb + c] = v;
        else if (c < g.d) g.F[(int64_t)e * g.d + c] = v;
    }
#endif
}

// Adds the slots of the groups that were cut, in chunk order.  One workgroup per (group, block pair).
__global__ __launch_bounds__(256) void grouped_gram_reduce_kernel(GramArgs g) {
    const int e = blockIdx.x / g.pairs, pair = blockIdx.x - e * g.pairs;
    const int64_t s0 = g.slots[e], s1 = g.slots[e + 1];
    if (s0 == s1) return;
    int bi, bj;
    pair_of(pair, g.nb, bi, bj);
    double* C = g.C + (int64_t)e * g.d * g.d;
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    for (int64_t s = s0; s < s1; ++s) {
        const double* p = g.part + (s * g.pairs + pair) * 1024 + threadIdx.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += p[256 * i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int el = threadIdx.x + 256 * i, r = 32 * bi + (el >> 5), c = 32 * bj + (el & 31);
        if (r <= c && c < g.d) {
            C[(int64_t)r * g.d + c] = v[i];
            if (r < c) C[(int64_t)c * g.d + r] = v[i];
        }
    }
    if (bi == bj && threadIdx.x < 32) {
        const int c = 32 * bi + threadIdx.x;
        double f = 0.0;
        for (int64_t s = s0; s < s1; ++s) f += g.part_f[s * 32 * g.nb + c];
        if (c < g.d) g.F[(int64_t)e * g.d + c] = f;
    }
}

}  // namespace hypmi_detail

using namespace hypmi_detail;

extern "C" int hypmi_grouped_gram_span(void) { return GRAM_SPAN; }

extern "C" int64_t hypmi_grouped_gram_workspace_bytes(int64_t n_slots, int d) {
    if (n_slots <= 0 || d <= 0) return 0;
    const int64_t nb = (d + 31) / 32;
    return n_slots * (nb * (nb + 1) / 2 * 1024 + 32 * nb) * 8;
}

extern "C" int hypmi_grouped_gram_f64(const void* x, int x_type, int64_t ldx, int d, const double* w,
                                      const int64_t* offsets, const int64_t* chunks, const int64_t* slots,
                                      int n_groups, int64_t n_chunks, int64_t n_slots, const int32_t* order, double* C,
                                      double* F, void* workspace, int64_t workspace_bytes, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    HYPMI_REQUIRE(n_groups >= 0 && n_chunks >= 0 && n_slots >= 0 && d > 0, "grouped_gram: bad shape");
    HYPMI_REQUIRE(x_type == HYPMI_F32 || x_type == HYPMI_F64, "grouped_gram: vectors must be fp32 or fp64");
    HYPMI_REQUIRE(ldx >= d, "grouped_gram: bad leading dimension");
    if (n_groups == 0) return HYPMI_OK;
    HYPMI_REQUIRE(offsets && chunks && slots && C && F, "grouped_gram: null pointer");
    HYPMI_REQUIRE(n_chunks >= n_groups, "grouped_gram: every group has a chunk");
    HYPMI_REQUIRE(workspace_bytes >= hypmi_grouped_gram_workspace_bytes(n_slots, d) && (n_slots == 0 || workspace),
                  "grouped_gram: workspace too small");
    const int nb = (d + 31) / 32;
    HYPMI_REQUIRE(nb <= 2048, "grouped_gram: more than 65536 features");
    const int pairs = nb * (nb + 1) / 2;
    double* part = static_cast<double*>(workspace);
    const GramArgs g = {x, ldx, d, w, offsets, chunks, slots, n_groups, n_chunks, order, C, F, part,
                        part ? part + n_slots * pairs * 1024 : nullptr, nb, pairs};
    const int64_t grid = xcd_grid(n_chunks * ((pairs + 3) / 4));
    const int64_t reduce = n_slots ? (int64_t)n_groups * pairs : 0;
    HYPMI_REQUIRE(grid <= 0x7fffffffLL && reduce <= 0x7fffffffLL, "grouped_gram: too many workgroups");
    if (x_type == HYPMI_F32)
        hipLaunchKernelGGL(grouped_gram_kernel<float>, dim3((unsigned)grid), dim3(256), 0, stream, g);
    else
        hipLaunchKernelGGL(grouped_gram_kernel<double>, dim3((unsigned)grid), dim3(256), 0, stream, g);
    HYPMI_HIP(hipGetLastError());
    if (reduce) {
        hipLaunchKernelGGL(grouped_gram_reduce_kernel, dim3((unsigned)reduce), dim3(256), 0, stream, g);
        HYPMI_HIP(hipGetLastError());
    }
    return HYPMI_OK;
}
