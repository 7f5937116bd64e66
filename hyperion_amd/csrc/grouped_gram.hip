// Grouped second-order moments  C_e = sum_r w_r x_r x_r^T,  F_e = sum_r w_r x_r  over the rows r of every
// group e, in float64: the covariance of every recording of a batch (the per-recording PCA of
// hyperion/diarization/diar_ahc_plda.py:131-141, whose statistics are np.dot(x.T, x),
// hyperion/pdfs/core/normal.py:102-113) or of every domain of a training set, in one pass.
//
// What bounds it is the float64 matrix instruction: v_mfma_f64_16x16x4 sustains 70 TFLOP/s over registers on this
// chip (v_fma_f64 55 to 60, with or without row broadcasts; both together no more than either).  A wave owns a
// 32 x 32 block of C; an operand is four samples of sixteen features, read as it lies in memory: four 8-byte loads
// per lane feed four instructions of 64 clocks, without shared memory.  Sixteen samples are in flight while the
// sixteen before them are multiplied.  Only blocks on or above the diagonal are computed (and three quarters of
// those on it), and both halves are written from them.
//
// Groups differ in size by orders of magnitude, and a wave with a thousand rows runs for 25 us: a chunk of more than
// GRAM_SPLIT rows is therefore shared by the four waves of a workgroup, a quarter each, which add their blocks in
// shared memory; in smaller ones every wave has a block of its own.  A group of more than GRAM_SPAN rows is cut into
// chunks of one length; every chunk writes its block to a slot of the workspace and a second kernel adds the slots in
// chunk order.  No sum depends on scheduling.
//
// Measured: 57 300 float64 rows of 7 groups, d = 512, 317 us back to back, 14 of them the second kernel (47.5 TFLOP/s);
// 25 600 fp32 rows of 200 groups, d = 200, 45 us, of which the matrix instructions are 20 and the writing of 64 MB 13.
// GRAM_SPLIT: with 200 groups of 96 rows a wave per block takes 32 us and four waves 44, with 384 and more rows 47 to
// 60 and 50 to 48; the ragged groups above take 50.3 / 48.9 / 49.9 / 51.6 / 53.2 us with a limit of 128 / 192 / 256 /
// 320 / 400 rows.  GRAM_SPAN of 1024 / 1536 / 2048 / 4096 rows, the mean of three sets of sizes in us: float64, d = 512, 7
// groups 336 / 331 / 329 / 331; d = 200, 3 groups 136 / 133 / 137 / 148; fp32, d = 200, 7 groups 78 / 77 / 76 / 88;
// d = 150, 20 groups 56 / 57 / 60 / 69; one group of 30 000 rows, d = 128, 43 / 33 / 35 / 47.  From 1536 to 2048 the sizes
// of the groups decide, 4096 leaves too few chunks, 1024 adds a slot per chunk to write and read again.
#include "grouped.h"

#include <type_traits>

namespace hypmi_detail {

struct GramArgs {
    const void* x;
    int64_t ldx;
    int d;
    const double* w;
    const int64_t* offsets;
    const int64_t* units;   // [n_groups + 1] prefix of the units of work: four for a shared chunk, one for a small one
    const int64_t* slots;   // [n_groups + 1] prefix of the number of chunks of groups that have several, 0 for the others
    int n_groups;
    int64_t n_units;
    const int32_t* order;
    double* C;
    double* F;
    double* part;           // [slots][pairs][32 * 32], then [slots][32 nb]
    double* part_f;
    int nb, pairs;
};

constexpr int GRAM_SPAN = 2048;  // rows of one chunk at most
constexpr int GRAM_SPLIT = 192;  // a chunk of more rows is shared by four waves

typedef double f64x4 __attribute__((ext_vector_type(4)));

// block pair p (row-major over bi <= bj) -> bi, bj
__device__ __forceinline__ void pair_of(int p, int nb, int& bi, int& bj) {
    bi = 0;
    while (p >= nb - bi) {
        p -= nb - bi;
        ++bi;
    }
    bj = bi + p;
}

// Four steps of four samples; `a` / `b` are the row and the column side of the block.
template <typename XT>
struct GramBatch {
    XT a[4][2], b[4][2];
    double w[4];
};

template <typename XT, bool ORDERED, bool WEIGHTED>
__global__ __launch_bounds__(256, 2) void grouped_gram_kernel(GramArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
    // [wave][tile][16][17] while a chunk's blocks are added up, the first 16 x 17 of a wave's part to turn a tile
    __shared__ double sums[4][4][16][17];
    __shared__ double sums_f[4][2][16];
    const int quads = (g.pairs + 3) >> 2;
    const int64_t t = xcd_task(blockIdx.x, g.n_units * quads, quads);
    if (t < 0) return;
    const int64_t unit = t / quads;
    const int quad = (int)(t - unit * quads);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int e = find_group(g.units, g.n_groups, unit);
    const int64_t u0 = unit - g.units[e], s_lim = g.offsets[e + 1], size = s_lim - g.offsets[e];
    // all chunks but the last have four units each; the chunks of a group are of one length
    const int64_t ch = u0 >> 2, cut = size > GRAM_SPAN ? (size + GRAM_SPAN - 1) / GRAM_SPAN : 1;
    const int64_t span = ((size + cut - 1) / cut + 63) & ~63LL;  // at most GRAM_SPAN where cut > 1
    int64_t s_beg = g.offsets[e] + ch * span;
    int ns = s_lim - s_beg < span ? (int)(s_lim - s_beg) : (int)span;
    const bool split = ns > GRAM_SPLIT;
    const int pair = quad * 4 + (split ? (int)(u0 & 3) : wave);
    if (pair >= g.pairs) return;  // the whole workgroup where the chunk is shared
    int bi, bj;
    pair_of(pair, g.nb, bi, bj);
    if (split) {
        const int part = ((ns + 63) >> 6) << 4;  // a quarter, in batches of sixteen
        const int from = wave * part < ns ? wave * part : ns;
        ns = ns - from < part ? ns - from : part;
        s_beg += from;
    }
    const bool diag = bi == bj;
    const int lane = threadIdx.x & 63, l15 = lane & 15, l4 = lane >> 4;
    const XT* X = static_cast<const XT*>(g.x);
    unsigned fa[2], fb[2];  // features of this lane, clamped into the row: those past it are computed and not stored
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int u = 32 * bi + 16 * h + l15, v = 32 * bj + 16 * h + l15;
        fa[h] = (unsigned)(u < g.d ? u : g.d - 1);
        fb[h] = (unsigned)(v < g.d ? v : g.d - 1);
    }
    f64x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = (f64x4){0.0, 0.0, 0.0, 0.0};
    double f[2] = {0.0, 0.0};

    // samples s .. s + 15 of the chunk; in the last batch a sample past the end is a copy of the last one
    auto fetch = [&](GramBatch<XT>& v, int s, bool last) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            int r = s + 4 * k + l4;
            if (last && r >= ns) r = ns - 1;
            if constexpr (ORDERED) {
                const int64_t row = g.order[s_beg + r];
                const XT* p = X + row * g.ldx;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    v.a[k][h] = p[fa[h]];
                    v.b[k][h] = p[fb[h]];
                }
                if (WEIGHTED) v.w[k] = g.w[row];
            } else {
                const XT* p = X + (s_beg + s + 4 * k) * g.ldx;  // the same for all lanes
                const int64_t d = (int64_t)(r - s - 4 * k) * g.ldx;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    v.a[k][h] = p[d + fa[h]];
                    v.b[k][h] = p[d + fb[h]];
                }
                if (WEIGHTED) v.w[k] = g.w[s_beg + r];
            }
        }
    };
    auto walk = [&](auto diag_tag) {
        constexpr bool DIAG = decltype(diag_tag)::value;
        auto multiply = [&](const GramBatch<XT>& v, int s, bool last) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                double da[2], db[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    da[h] = (double)v.a[k][h];
                    db[h] = (double)v.b[k][h];
                    if (WEIGHTED) db[h] *= v.w[k];
                    if (last && s + 4 * k + l4 >= ns) da[h] = db[h] = 0.0;
                    if (DIAG) f[h] += db[h];
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        if (i <= j || !DIAG)
                            acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(da[i], db[j], acc[i][j], 0, 0, 0);
            }
        };
        // two batches by turns, so that none is copied: a copy would wait for its loads before the batch at hand
        // is multiplied
        GramBatch<XT> u, v;
        int s = 0;
        if (ns >= 16) fetch(u, 0, false);
        for (; s + 32 <= ns; s += 32) {
            fetch(v, s + 16, false);
            __builtin_amdgcn_sched_barrier(0);
            multiply(u, s, false);
            __builtin_amdgcn_sched_barrier(0);
            fetch(u, s + 48 <= ns ? s + 32 : s, false);  // always as many loads: the waits are counted
            __builtin_amdgcn_sched_barrier(0);
            multiply(v, s + 16, false);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (s + 16 <= ns) {
            multiply(u, s, false);
            s += 16;
        }
        if (s < ns) {
            fetch(v, s, true);
            multiply(v, s, true);
        }
    };
    if (diag) walk(std::true_type{});
    else walk(std::false_type{});
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        f[h] += __shfl_xor(f[h], 16);
        f[h] += __shfl_xor(f[h], 32);
    }
    const int64_t slot = size > GRAM_SPAN ? g.slots[e] + ch : -1;
    double* part = g.part + (slot * g.pairs + pair) * 1024;
    double* C = g.C + (int64_t)e * g.d * g.d;
    // tile (i, j) of the block, lane: rows l4 + 4 q, column l15
    auto write = [&](int i, int j, const f64x4& v) {
        const int r0 = 32 * bi + 16 * i, c0 = 32 * bj + 16 * j;
        if (slot >= 0) {
#pragma unroll
            for (int q = 0; q < 4; ++q) part[(16 * i + l4 + 4 * q) * 32 + 16 * j + l15] = v[q];
            return;
        }
        double(*turn)[17] = sums[wave][split ? i * 2 + j : 0];  // this wave's own until the end
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = r0 + l4 + 4 * q, c = c0 + l15;
            if (r <= c && c < g.d) C[(int64_t)r * g.d + c] = v[q];
            turn[l15][l4 + 4 * q] = v[q];
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // the other half: rows of the transposed tile
            const int c = c0 + l4 + 4 * q, r = r0 + l15;
            if (r < c && c < g.d) C[(int64_t)c * g.d + r] = turn[l4 + 4 * q][l15];
        }
        __builtin_amdgcn_wave_barrier();
    };
    auto write_f = [&](double v, int h) {  // 16 lanes: feature 32 bi + 16 h + l15
        const int c = 32 * bi + 16 * h + l15;
        if (slot >= 0) g.part_f[slot * 32 * g.nb + c] = v;
        else if (c < g.d) g.F[(int64_t)e * g.d + c] = v;
    };
    if (split) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) sums[wave][i * 2 + j][l4 + 4 * q][l15] = acc[i][j][q];
        if (diag && l4 < 2) sums_f[wave][l4][l15] = l4 ? f[1] : f[0];
        __syncthreads();
        f64x4 v;  // wave w finishes tile w
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            v[q] = sums[0][wave][l4 + 4 * q][l15];
#pragma unroll
            for (int w = 1; w < 4; ++w) v[q] += sums[w][wave][l4 + 4 * q][l15];
        }
        double fs = 0.0;
        if (diag && wave < 2 && l4 == 0) {
#pragma unroll
            for (int w = 0; w < 4; ++w) fs += sums_f[w][wave][l15];
        }
        __syncthreads();  // `write` turns tiles in the same memory
        if (!diag || wave != 2) write(wave >> 1, wave & 1, v);
        if (diag && wave < 2 && l4 == 0) write_f(fs, wave);
        return;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (i <= j || !diag) write(i, j, acc[i][j]);
    if (diag && l4 < 2) write_f(l4 ? f[1] : f[0], l4);
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
extern "C" int hypmi_grouped_gram_split(void) { return GRAM_SPLIT; }

extern "C" int64_t hypmi_grouped_gram_workspace_bytes(int64_t n_slots, int d) {
    if (n_slots <= 0 || d <= 0) return 0;
    const int64_t nb = (d + 31) / 32;
    return n_slots * (nb * (nb + 1) / 2 * 1024 + 32 * nb) * 8;
}

extern "C" int hypmi_grouped_gram_f64(const void* x, int x_type, int64_t ldx, int d, const double* w,
                                      const int64_t* offsets, const int64_t* units, const int64_t* slots,
                                      int n_groups, int64_t n_units, int64_t n_slots, const int32_t* order, double* C,
                                      double* F, void* workspace, int64_t workspace_bytes, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    HYPMI_REQUIRE(fits_groups(n_groups) && n_units >= 0 && n_slots >= 0 && d > 0, "grouped_gram: bad shape");
    HYPMI_REQUIRE(x_type == HYPMI_F32 || x_type == HYPMI_F64, "grouped_gram: vectors must be fp32 or fp64");
    HYPMI_REQUIRE(ldx >= d, "grouped_gram: bad leading dimension");
    if (n_groups == 0) return HYPMI_OK;
    HYPMI_REQUIRE(offsets && units && slots && C && F, "grouped_gram: null pointer");
    HYPMI_REQUIRE(n_units >= n_groups, "grouped_gram: every group has a unit of work");
    HYPMI_REQUIRE(workspace_bytes >= hypmi_grouped_gram_workspace_bytes(n_slots, d) && (n_slots == 0 || workspace),
                  "grouped_gram: workspace too small");
    const int nb = (d + 31) / 32;
    HYPMI_REQUIRE(nb <= 2048, "grouped_gram: more than 65536 features");
    const int pairs = nb * (nb + 1) / 2;
    double* part = static_cast<double*>(workspace);
    const GramArgs g = {x, ldx, d, w, offsets, units, slots, n_groups, n_units, order, C, F, part,
                        part ? part + n_slots * pairs * 1024 : nullptr, nb, pairs};
    HYPMI_REQUIRE(fits_launch(n_units, 256), "grouped_gram: too many units of work");  // below 2^24: no product overflows
    const int64_t grid = xcd_grid(n_units * ((pairs + 3) / 4), (pairs + 3) / 4);
    const int64_t reduce = n_slots ? (int64_t)n_groups * pairs : 0;
    HYPMI_REQUIRE(fits_launch(grid, 256) && fits_launch(reduce, 256), "grouped_gram: too many workgroups");
    const dim3 blocks((unsigned)grid), threads(256);
    auto launch = [&](auto type, auto ordered) {
        typedef decltype(type) XT;
        constexpr bool O = decltype(ordered)::value;
        if (w) hipLaunchKernelGGL((grouped_gram_kernel<XT, O, true>), blocks, threads, 0, stream, g);
        else hipLaunchKernelGGL((grouped_gram_kernel<XT, O, false>), blocks, threads, 0, stream, g);
    };
    if (x_type == HYPMI_F32) order ? launch(float(), std::true_type{}) : launch(float(), std::false_type{});
    else order ? launch(double(), std::true_type{}) : launch(double(), std::false_type{});
    HYPMI_HIP(hipGetLastError());
    if (reduce) {
        hipLaunchKernelGGL(grouped_gram_reduce_kernel, dim3((unsigned)reduce), dim3(256), 0, stream, g);
        HYPMI_HIP(hipGetLastError());
    }
    return HYPMI_OK;
}
