// Grouped score blocks  S_e = G1_e G2_e^T  from packed rows: for every group e the log-likelihood ratios of
// its enrol-side rows against its test-side rows (hypmi_score per recording or domain; the self-scores of
// hyperion/diarization/diar_ahc_plda.py:141-143 for a whole batch of recordings in one launch).  Blocks are
// stored one after the other without padding, block e row-major [n1_e x n2_e] at block_offsets[e].
//
// Arithmetic as in score_split.hip: every row is scaled by a power of two and written as a pair of fp16
// numbers, three of the four partial products are accumulated in fp32 on the fp16 matrix cores.  The rows
// are converted here, on their way to the matrix instructions: a block has only as many columns as the group
// has rows, so a converted copy of the operands would cost as much traffic as the scores themselves.
//
// A wave keeps 16 RT enrol rows as operands in registers and walks up to `span` test rows of its group in tiles of
// 32 (a group's test rows are cut into equal parts), which the four waves of the workgroup load, convert (a row's
// largest magnitude over eight lanes) and leave in LDS in operand order; the values of the next two tiles are in
// flight meanwhile.  Test rows are the first operand of the matrix instruction, so a lane ends up with four
// neighbouring scores of one enrol row.
//
// Measured at a packed width of 152: 200 recordings of 12 to 900 segments (16.2 M scores) 42 us, 12 domains of 300 to
// 20000 test vectors (68.9 M scores) 120 to 135 us: 2.0 to 2.3 TB/s of results, 0.5 PFLOP/s of fp16 products.  What
// bounds it is the issue of instructions: of a tile's 3600 clocks per wave 960 are matrix instructions and 900 vector
// ones, and two waves per SIMD hide little of either behind the other.  Without the matrix instructions the domains
// take 53 us, without the stores 95, without the conversion 5 less; spans of 256 to 768, three waves per SIMD, tiles
// fetched one or three ahead and stores of whole lines stay within 5 % of this.
#include "grouped.h"

#include <type_traits>

namespace hypmi_detail {

struct ScoreArgs {
    const float* G1;
    const float* G2;
    int64_t ld1, ld2;
    int kp;
    const int64_t* off1;    // [n_groups + 1]
    const int64_t* off2;
    const int64_t* blocks;  // [n_groups + 1] element offsets of the blocks
    const int64_t* tasks;   // [n_groups + 1] prefix of ceil(n1 / (64 RT)) * ceil(n2 / span)
    int n_groups;
    int64_t n_tasks;
    int span;
    float* S;
};

constexpr int SCORE_RUN = 8;     // tasks dealt to an XCD at a time
constexpr int SCORE_SPAN = 512;  // test rows one workgroup walks at most

template <int KS, int RT>  // k-steps of 32 coordinates, row tiles of 16 per wave
__global__ __launch_bounds__(256) void grouped_score_kernel(ScoreArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr int OCT = (4 * KS + 7) / 8;  // octets of coordinates per lane of the loading side
    __shared__ uint4 tile[2][2 * KS * 2 * 64];  // [buffer][(column tile, k-step, part, lane)]
    __shared__ int scale[2][32];

    const int64_t t = xcd_task(blockIdx.x, g.n_tasks, SCORE_RUN);
    if (t < 0) return;
    const int e = find_group(g.tasks, g.n_groups, t);
    const int64_t n1 = g.off1[e + 1] - g.off1[e], n2 = g.off2[e + 1] - g.off2[e];
    const int64_t spans = (n2 + g.span - 1) / g.span;
    const int64_t task = t - g.tasks[e];
    const int64_t i_blk = task / spans;
    const int64_t span = ((n2 + spans - 1) / spans + 31) & ~31LL;  // equal parts, at most g.span
    const int64_t j_beg = (task - i_blk * spans) * span;
    const int ncol = n2 - j_beg < span ? (int)(n2 - j_beg) : (int)span;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    const float* G2 = g.G2 + (g.off2[e] + j_beg) * g.ld2;

    // ---- test side: lane loads octets (lane >> 3) + 8 o of row 8 wave + (lane & 7) of a tile
    const int lr = 8 * wave + (lane & 7), lo = lane >> 3;
    typedef f32x4 Octets[OCT][2];
    Octets v, u;
    // Every call issues the same loads, so that the waits for one tile's values are counted past those of the next
    // and past stores: behind the last row the last row is read again, behind the last octet the last octet (taken
    // out by value in `store`).
    int oct_at[OCT];
#pragma unroll
    for (int o = 0; o < OCT; ++o) oct_at[o] = 8 * (lo + 8 * o) < g.kp ? 8 * (lo + 8 * o) : g.kp - 8;
    auto fetch = [&](Octets& v, int tile) {
        const int j = 32 * tile + lr < ncol ? 32 * tile + lr : ncol - 1;
        const float* p = G2 + j * g.ld2;
#pragma unroll
        for (int o = 0; o < OCT; ++o) {
            v[o][0] = *reinterpret_cast<const f32x4*>(p + oct_at[o]);
            v[o][1] = *reinterpret_cast<const f32x4*>(p + oct_at[o] + 4);
        }
    };
    auto store = [&](const Octets& v, int buf) {
        float m = 0.f;
#pragma unroll
        for (int o = 0; o < OCT; ++o)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < 4; ++q) m = fmaxf(m, fabsf(v[o][h][q]));
#pragma unroll
        for (int x = 8; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x));
        int up = m > 0.f ? 15 - __builtin_amdgcn_frexp_expf(m) : 0;
        up = up > 126 ? 126 : up;
        if (lo == 0) scale[buf][lr] = up;
        const float f = exp2_int(up);
        const int ct = lr >> 4, row = lr & 15;
#pragma unroll
        for (int o = 0; o < OCT; ++o) {
            const int oct = lo + 8 * o;
            if (oct >= 4 * KS) continue;
            const float fo = 8 * oct < g.kp ? f : 0.f;
            const int s = oct >> 2, q = oct & 3;
            f16x4 a0, a1, b0, b1;
            split_pair4(v[o][0], fo, a0, a1);
            split_pair4(v[o][1], fo, b0, b1);
            f16x4* dst = reinterpret_cast<f16x4*>(&tile[buf][((ct * KS + s) * 2) * 64 + q * 16 + (row ^ (8 * (q & 1)))]);
            dst[0] = a0;
            dst[1] = b0;
            dst[128] = a1;
            dst[129] = b1;
        }
    };

    fetch(v, 0);
    fetch(u, 1);
    __builtin_amdgcn_sched_barrier(0);

    // ---- enrol side: a[i][s][part] = coordinates 32 s + 8 kq .. + 7 of row i0 + 16 i + r16
    const int64_t i0 = (i_blk * 4 + wave) * (16 * RT);
    f16x8 a[RT][KS][2];
    int rs[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        int64_t row = i0 + 16 * i + r16;
        row = row < n1 ? row : n1 - 1;
        const float* p = g.G1 + (g.off1[e] + row) * g.ld1 + 8 * kq;
        f32x4 x[KS][2];
        float m = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (32 * s + 8 * kq < g.kp) {
                x[s][0] = *reinterpret_cast<const f32x4*>(p + 32 * s);
                x[s][1] = *reinterpret_cast<const f32x4*>(p + 32 * s + 4);
            } else {
                x[s][0] = x[s][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < 4; ++q) m = fmaxf(m, fabsf(x[s][h][q]));
        }
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        int up = m > 0.f ? 15 - __builtin_amdgcn_frexp_expf(m) : 0;
        up = up > 126 ? 126 : up;
        rs[i] = up;
        const float f = exp2_int(up);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            f16x4 a0, a1, b0, b1;
            split_pair4(x[s][0], f, a0, a1);
            split_pair4(x[s][1], f, b0, b1);
            a[i][s][0] = __builtin_shufflevector(a0, b0, 0, 1, 2, 3, 4, 5, 6, 7);
            a[i][s][1] = __builtin_shufflevector(a1, b1, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    const int xs = kq * 16 + (r16 ^ (8 * (kq & 1)));
    // result rows of this lane; a row past the end holds the last row's scores (its operand is a copy) and stores
    // them to the same place, so that no store depends on a comparison
    float* dst[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t row = i0 + 16 * i + r16;
        dst[i] = g.S + g.blocks[e] + (row < n1 ? row : n1 - 1) * n2 + j_beg + 4 * kq;
    }
    auto multiply = [&](int it, bool whole) {
        const int buf = it & 1;
        f32x4 acc[RT][2];
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i][0] = acc[i][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint4* p = &tile[buf][((c * KS + s) * 2) * 64 + xs];
                const f16x8 b0 = __builtin_bit_cast(f16x8, p[0]);
                const f16x8 b1 = __builtin_bit_cast(f16x8, p[64]);
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b1, a[i][s][0], acc[i][c], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b0, a[i][s][1], acc[i][c], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b0, a[i][s][0], acc[i][c], 0, 0, 0);
            }
        // lane: columns 32 it + 16 c + 4 kq .. + 3 of enrol row i0 + 16 i + r16
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int j = 32 * it + 16 * c;
            const int4 cs = *reinterpret_cast<const int4*>(&scale[buf][16 * c + 4 * kq]);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                // one shift by the sum of both exponents: neither scale alone may leave the range
                const f32x4 r = {ldexpf(acc[i][c][0], -rs[i] - cs.x), ldexpf(acc[i][c][1], -rs[i] - cs.y),
                                 ldexpf(acc[i][c][2], -rs[i] - cs.z), ldexpf(acc[i][c][3], -rs[i] - cs.w)};
                if (whole) {
                    *reinterpret_cast<f32x4_a4*>(dst[i] + j) = r;
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (j + 4 * kq + q < ncol) dst[i][j + q] = r[q];
                }
            }
        }
    };

    auto walk = [&](auto live_tag) {
        constexpr bool LIVE = decltype(live_tag)::value;  // this wave has rows
        store(v, 0);
        fetch(v, 2);
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        const int whole = ncol >> 5;
        for (int it = 0; it < whole; it += 2) {
            if (LIVE) multiply(it, true);
            store(u, 1);
            fetch(u, it + 3);
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
            if (it + 1 == whole) break;
            if (LIVE) multiply(it + 1, true);
            store(v, 0);
            fetch(v, it + 4);
            __builtin_amdgcn_sched_barrier(0);
            __syncthreads();
        }
        if (LIVE && 32 * whole < ncol) multiply(whole, false);
    };
    if (i0 < n1) walk(std::true_type{});
    else walk(std::false_type{});
#endif
}

template <int KS>
int launch_score(const ScoreArgs& g, hipStream_t stream) {
    constexpr int RT = KS <= 6 ? 2 : 1;
    const int64_t grid = xcd_grid(g.n_tasks, SCORE_RUN);
    HYPMI_REQUIRE(grid <= 0x7fffffffLL, "grouped_score: too many workgroups");
    hipLaunchKernelGGL((grouped_score_kernel<KS, RT>), dim3((unsigned)grid), dim3(256), 0, stream, g);
    HYPMI_HIP(hipGetLastError());
    return HYPMI_OK;
}

}  // namespace hypmi_detail

using namespace hypmi_detail;

extern "C" int hypmi_grouped_score_rows(int kp) {
    if (kp <= 0 || kp % 8 != 0 || kp > 512) return 0;
    return (kp + 31) / 32 <= 6 ? 128 : 64;
}

extern "C" int hypmi_grouped_score_span(void) { return SCORE_SPAN; }

extern "C" int hypmi_grouped_score(const float* G1, int64_t ld1, const float* G2, int64_t ld2, int kp,
                                   const int64_t* offsets1, const int64_t* offsets2, const int64_t* block_offsets,
                                   const int64_t* tasks, int n_groups, int64_t n_tasks, float* S, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    HYPMI_REQUIRE(n_groups >= 0 && n_tasks >= 0, "grouped_score: bad shape");
    HYPMI_REQUIRE(hypmi_grouped_score_rows(kp) > 0, "grouped_score: packed width %d (a multiple of 8 up to 512)", kp);
    HYPMI_REQUIRE(ld1 >= kp && ld2 >= kp && ld1 % 4 == 0 && ld2 % 4 == 0, "grouped_score: bad leading dimension");
    if (n_tasks == 0) return HYPMI_OK;
    HYPMI_REQUIRE(G1 && G2 && offsets1 && offsets2 && block_offsets && tasks && S, "grouped_score: null pointer");
    HYPMI_REQUIRE(aligned16(G1) && aligned16(G2), "grouped_score: packed rows must be 16-byte aligned");
    const ScoreArgs g = {G1, G2, ld1, ld2, kp, offsets1, offsets2, block_offsets, tasks, n_groups, n_tasks, SCORE_SPAN, S};
    switch ((kp + 31) / 32) {
        case 1: return launch_score<1>(g, stream);
        case 2: return launch_score<2>(g, stream);
        case 3: return launch_score<3>(g, stream);
        case 4: return launch_score<4>(g, stream);
        case 5: return launch_score<5>(g, stream);
        case 6: return launch_score<6>(g, stream);
        case 7: return launch_score<7>(g, stream);
        case 8: return launch_score<8>(g, stream);
        case 9:
        case 10: return launch_score<10>(g, stream);
        case 11:
        case 12: return launch_score<12>(g, stream);
        default: return launch_score<16>(g, stream);
    }
}
