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
// A workgroup has four or eight waves that multiply and two that load.  A multiplying wave keeps 16 enrol rows as
// operands in registers and walks up to `span` test rows of its group in tiles of 32 (a group's test rows are cut into
// equal parts); the loading waves take 16 rows of the next tile each, a row by four lanes, find its largest magnitude,
// convert it and leave it in LDS in operand order, and request the tile after that.  Memory operations of a wave
// complete in order, so a wave that both stores scores and loads rows waits for its scores to be written: with four
// waves that did both, 200 recordings took 42 us instead of 35; the 12 domains gained little (117 instead of 107 at best
// for the kernel alone, nothing for passes that follow one another).  Test rows
// are the first operand of the matrix instruction, so a lane ends up with four neighbouring scores of one enrol row.
//
// Measured at a packed width of 152: 200 recordings of 12 to 900 segments (16.2 M scores) 33 to 40 us from card to card, 12
// domains of 300 to 20000 test vectors (68.9 M scores) 136, of which the kernel alone 107 to 126 after a pause: 2.0 TB/s
// of results.  The domains write 334 MB for 276 (a row of a block starts anywhere in a line) and read 91 MB for 20;
// without the stores they take 95 us, with the stores and one multiplication per span 76 to 85, so neither alone is the
// bound: 1152 workgroups, two per CU, are 2.25 rounds, and a loading wave has one tile in flight.  Enrol blocks in
// turn instead of spans read 47 MB but leave the last workgroups alone for longer (114 us at best); spans of 256 to
// 1024, 32 rows a wave (109 us), rows converted beforehand by a kernel of their own (131 + 10 us) are not faster.
#include "grouped.h"

namespace hypmi_detail {

struct ScoreArgs {
    const float* G1;
    const float* G2;
    int64_t ld1, ld2;
    int kp;
    const int64_t* off1;    // [n_groups + 1]
    const int64_t* off2;
    const int64_t* blocks;  // [n_groups + 1] element offsets of the blocks
    const int64_t* tasks;   // [n_groups + 1] prefix of ceil(n1 / (16 NW)) * ceil(n2 / span)
    int n_groups;
    int64_t n_tasks;
    int span;
    float* S;
};

constexpr int SCORE_RUN = 8;     // tasks dealt to an XCD at a time
constexpr int SCORE_SPAN = 512;  // test rows one workgroup walks at most

// Multiplying waves of a workgroup, 16 enrol rows each.  Recordings (17.5 M scores) / domains (12.5 M) with eight
// waves, with four, with four that take 32 rows each, in us: 3 k-steps 35 / 23, 39 / 27, 35 / 24; 5 k-steps 40 / 26, 46 / 30,
// 40 / 27; 6 k-steps 53 / 32, 63 / 39, 62 / 34.  Eight would be faster above 192 columns too (8 k-steps 74 / 39 against
// 85 / 56, 16 k-steps 144 / 72 against 160 / 103), where callers count their tasks in 64 rows.
constexpr int score_waves(int ksteps) { return ksteps <= 6 ? 8 : 4; }

// Coordinates 32 s + 8 kq .. + 7 of the row at `p`, s = 0 .. KS - 1; lanes r16 + 16 kq hold one row.  Past the end of a
// row its last octet is read again, taken out by value in `operand`.
template <int KS>
struct RowValues {
    f32x4 x[KS][2];

    __device__ __forceinline__ void fetch(const float* p, int kp, int kq) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int k = 32 * s + 8 * kq, at = k < kp ? k : kp - 8;
            x[s][0] = *reinterpret_cast<const f32x4*>(p + at);
            x[s][1] = *reinterpret_cast<const f32x4*>(p + at + 4);
        }
    }

    // exponent of the power of two that takes the row's largest magnitude to [2^14, 2^15)
    __device__ __forceinline__ int scale() const {
        float m = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < 4; ++q) m = fmaxf(m, fabsf(x[s][h][q]));
        m = swap32_max(swap16_max(m));
        const int up = m > 0.f ? 15 - __builtin_amdgcn_frexp_expf(m) : 0;
        return up > 126 ? 126 : up;
    }

    __device__ __forceinline__ void operand(int s, float f, int kp, int kq, f16x8& a0, f16x8& a1) const {
        const float fs = 32 * s + 8 * kq < kp ? f : 0.f;
        f16x4 l0, l1, h0, h1;
        split_pair4(x[s][0], fs, l0, l1);
        split_pair4(x[s][1], fs, h0, h1);
        a0 = __builtin_shufflevector(l0, h0, 0, 1, 2, 3, 4, 5, 6, 7);
        a1 = __builtin_shufflevector(l1, h1, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// KS k-steps of 32 coordinates, NW multiplying waves.  The waves per SIMD asked for are those of two workgroups on a CU, of
// one above 256 columns, where its tiles fill more than half of the shared memory.
template <int KS, int NW>
__global__ __launch_bounds__(64 * NW + 128, NW == 8 ? 5 : KS <= 8 ? 3 : 2) void grouped_score_kernel(ScoreArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
    __shared__ uint4 tile[2][2 * KS * 2 * 64];  // [buffer][(column tile, k-step, part, lane)]
    __shared__ __attribute__((aligned(16))) int scale[2][32];

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
    const int tiles = (ncol + 31) >> 5;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;

    if (wave >= NW) {
        // ---- a loading wave: rows 16 c .. + 15 of every tile
        const int c = wave - NW;
        const float* G2 = g.G2 + (g.off2[e] + j_beg) * g.ld2;
        RowValues<KS> v;
        auto fetch = [&](int it) {
            const int j = 32 * it + 16 * c + r16;
            v.fetch(G2 + (int64_t)(j < ncol ? j : ncol - 1) * g.ld2, g.kp, kq);
        };
        auto store = [&](int buf) {
            const int up = v.scale();
            if (kq == 0) scale[buf][16 * c + r16] = up;
            const float f = exp2_int(up);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                f16x8 a0, a1;
                v.operand(s, f, g.kp, kq, a0, a1);
                uint4* dst = &tile[buf][((c * KS + s) * 2) * 64 + lane];
                dst[0] = __builtin_bit_cast(uint4, a0);
                dst[64] = __builtin_bit_cast(uint4, a1);
            }
        };
        fetch(0);
        store(0);
        fetch(1);
        __syncthreads();
        for (int it = 0; it < tiles; ++it) {
            if (it + 1 < tiles) {
                store((it + 1) & 1);
                fetch(it + 2);
            }
            __syncthreads();
        }
        return;
    }

    // ---- enrol side: a[s][part] = coordinates 32 s + 8 kq .. + 7 of row i0 + r16
    const int64_t i0 = (i_blk * NW + wave) * 16;
    const bool live = i0 < n1;  // this wave has rows
    f16x8 a[KS][2];
    int rs = 0;
    // result row of this lane; a row past the end holds the last row's scores (its operand is a copy) and stores
    // them to the same place, so that no store depends on a comparison
    float* dst = nullptr;
    if (live) {
        int64_t row = i0 + r16;
        row = row < n1 ? row : n1 - 1;
        dst = g.S + g.blocks[e] + row * n2 + j_beg + 4 * kq;
        RowValues<KS> v;
        v.fetch(g.G1 + (g.off1[e] + row) * g.ld1, g.kp, kq);
        rs = v.scale();
        const float f = exp2_int(rs);
#pragma unroll
        for (int s = 0; s < KS; ++s) v.operand(s, f, g.kp, kq, a[s][0], a[s][1]);
    }
    auto multiply = [&](int it, bool whole) {
        const int buf = it & 1;
        f32x4 acc[2];
        acc[0] = acc[1] = (f32x4){0.f, 0.f, 0.f, 0.f};
        f16x8 b[2][2][2];  // [k-step parity][column tile][part]
        auto request = [&](int s) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int p = 0; p < 2; ++p)
                    b[s & 1][c][p] = __builtin_bit_cast(f16x8, tile[buf][((c * KS + s) * 2 + p) * 64 + lane]);
        };
        request(0);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s + 1 < KS) request(s + 1);
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    acc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(b[s & 1][c][p == 0], a[s][p == 1], acc[c], 0, 0, 0);
        }
        // lane: columns 32 it + 16 c + 4 kq .. + 3 of enrol row i0 + r16
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int j = 32 * it + 16 * c;
            const int4 cs = *reinterpret_cast<const int4*>(&scale[buf][16 * c + 4 * kq]);
            // one shift by the sum of both exponents: neither scale alone may leave the range
            const f32x4 r = {ldexpf(acc[c][0], -rs - cs.x), ldexpf(acc[c][1], -rs - cs.y),
                             ldexpf(acc[c][2], -rs - cs.z), ldexpf(acc[c][3], -rs - cs.w)};
            if (whole) {
                *reinterpret_cast<f32x4_a4*>(dst + j) = r;
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (j + 4 * kq + q < ncol) dst[j + q] = r[q];
            }
        }
    };
    __syncthreads();
    const int whole = ncol >> 5;
    for (int it = 0; it < whole; ++it) {
        if (live) multiply(it, true);
        __syncthreads();
    }
    if (whole < tiles) {
        if (live) multiply(whole, false);
        __syncthreads();
    }
#endif
}

template <int KS>
int launch_score(const ScoreArgs& g, hipStream_t stream) {
    constexpr int NW = score_waves(KS);
    const int64_t grid = xcd_grid(g.n_tasks, SCORE_RUN);
    HYPMI_REQUIRE(fits_launch(grid, 64 * NW + 128), "grouped_score: too many workgroups");
    hipLaunchKernelGGL((grouped_score_kernel<KS, NW>), dim3((unsigned)grid), dim3(64 * NW + 128), 0, stream, g);
    HYPMI_HIP(hipGetLastError());
    return HYPMI_OK;
}

}  // namespace hypmi_detail

using namespace hypmi_detail;

extern "C" int hypmi_grouped_score_rows(int kp) {
    if (kp <= 0 || kp % 8 != 0 || kp > 512) return 0;
    return 16 * score_waves((kp + 31) / 32);
}

extern "C" int hypmi_grouped_score_span(void) { return SCORE_SPAN; }

extern "C" int hypmi_grouped_score(const float* G1, int64_t ld1, const float* G2, int64_t ld2, int kp,
                                   const int64_t* offsets1, const int64_t* offsets2, const int64_t* block_offsets,
                                   const int64_t* tasks, int n_groups, int64_t n_tasks, float* S, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    HYPMI_REQUIRE(fits_groups(n_groups) && n_tasks >= 0, "grouped_score: bad shape");
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
