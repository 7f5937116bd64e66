// Enrolment gallery in 4 bits: the projected rows g of packed enrol-side rows [g, q, 1] held as signed 4-bit
// codes with one scale per 32 coordinates, and their scores against a few test-side rows
//   S[t, i] = sum_k c_ik s_i(k / 32) g_t[k] + q_i + (q_t + c)
// (the product of hyperion/pdfs/plda/splda.py:312-315 against a coarser copy of one side; q is kept in fp32).
//
// Format.  The scale of 32 coordinates is the smallest bfloat16 number s with 7 s >= the largest magnitude, a
// code the integer nearest to x / s, halves to even (|c| <= 7), stored as c + 8; an error of at most s / 2 per
// coordinate.  A group of coordinates that holds a NaN or an infinity gets a NaN scale, which makes every score
// of that row NaN.  Rows are stored in blocks of 64 (a group of the gallery starts a new block):
//   codes  [block][k-step of 32][lane 0..63] uint4: component u holds the eight codes of row 16 u + (lane & 15),
//          coordinates 32 ks + 8 (lane >> 4) + j, code j at bit 8 (j >> 2) + 4 ((j >> 1) & 1) + 16 (j & 1): the two
//          codes of an fp16 pair sixteen bits apart;
//   scales [block][k-step][16] ushort4: component u the scale of row 16 u + l;    q [block][64] fp32.
// At 150 coordinates a row takes 94 bytes (fp32: 608).
//
// Scoring is one pass over the gallery.  A lane turns four bytes into the eight-element operand of
// v_mfma_f32_16x16x32_f16: a nibble under the exponent of 1024 is the fp16 number 1024 + c (or 1024 + 16 c for the
// nibble above it), and one packed fp16 operation makes c - 8 of either, exactly.  (Left as the sub-normal number
// that the bare nibble is, without that operation, a code is multiplied exactly but added with ten bits less:
// 3e-6 of the sum of magnitudes instead of 1e-7, measured.)  Test rows are scaled by a power of two and held as
// fp16 pairs (see score_split.hip), so a score is the product with the row that the codes stand for, the
// coordinates of the test to 22 bits or to 2^-39 of its largest.
// The contraction of one instruction is one scale group: its result is multiplied by the scale and added up in
// fp32.
//
// Measured at 150 coordinates: one test against a million rows 24 us (93 MB, 3.9 TB/s of a copy's 4.95), 1000 tests
// 1.2 ms, 40 partitions of 500 to 30 000 rows with 0 to 40 tests each 13 us (two dependent reads and the
// preparation of the tests come before the first product).
#include "grouped.h"

namespace hypmi_detail {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int Q4_RUN = 8;        // tasks dealt to an XCD at a time
constexpr int Q4_BLOCK = 64;     // rows of a block

// One thread per (row slot, k-step).
__global__ __launch_bounds__(256) void q4_rows_kernel(const float* __restrict__ G, int64_t ld, int k, int ks_all,
                                                      const int64_t* __restrict__ offsets,
                                                      const int64_t* __restrict__ blocks, int n_groups,
                                                      int64_t n_blocks, unsigned* __restrict__ codes,
                                                      unsigned short* __restrict__ scales, float* __restrict__ q) {
    // a wave: the 64 rows of one block, one k-step
    const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t blk = u / ks_all;
    if (blk >= n_blocks) return;
    const int ks = (int)(u - blk * ks_all);
    const int e = find_group(blocks, n_groups, blk);
    const int slot = threadIdx.x & 63;
    const int64_t row = offsets[e] + (blk - blocks[e]) * Q4_BLOCK + slot;
    const bool in = row < offsets[e + 1];
    const float* src = G + (in ? row : offsets[e]) * ld;
    float x[32];
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const int c = 32 * ks + i;
        x[i] = (in && c < k) ? src[c] : 0.f;
        const float a = fabsf(x[i]);
        bad |= !(a <= 3.402823466e38f);
        top = fmaxf(top, a);
    }
    // smallest bfloat16 with 7 s >= top: 7 s is exact in fp32 (8 + 3 bits)
    unsigned sb = __float_as_uint(top / 7.f) >> 16;
    if (7.f * __uint_as_float(sb << 16) < top) ++sb;
    const float s = __uint_as_float(sb << 16);
    unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        float c = 0.f;
        if (!bad && s > 0.f) {
            const float r = x[i] / s;
            c = rintf(r);
            // a quotient that rounded onto a half: the remainder says on which side x lies
            if (fabsf(r - truncf(r)) == 0.5f) {
                const float rem = fmaf(-r, s, x[i]);
                if (rem != 0.f) c = rem > 0.f ? ceilf(r) : floorf(r);
            }
        }
        const unsigned code = (unsigned)((int)c + 8);
        const int j = i & 7;
        w[i >> 3] |= code << (8 * (j >> 2) + 4 * ((j >> 1) & 1) + 16 * (j & 1));
    }
    unsigned* dst = codes + ((blk * ks_all + ks) * 64 + (slot & 15)) * 4 + (slot >> 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i * 64] = w[i];
    scales[((blk * ks_all + ks) * 16 + (slot & 15)) * 4 + (slot >> 4)] = bad ? 0x7fc0 : (unsigned short)sb;
    if (ks == 0) q[blk * Q4_BLOCK + slot] = in ? src[k] : 0.f;
}

struct Q4Args {
    const uint4* codes;
    const uint2* scales;
    const float* q;
    const float* G;         // test-side packed rows [g, 1, q + c]
    int64_t ld;
    int k;
    const int64_t* off_t;   // [n_groups + 1] tests
    const int64_t* off_g;   // [n_groups + 1] gallery rows
    const int64_t* blk;     // [n_groups + 1] prefix of gallery blocks
    const int64_t* out;     // [n_groups + 1] element offsets of the score blocks
    const int64_t* tasks;   // [n_groups + 1] prefix of ceil(n / run_rows) * ceil(m / (16 TT))
    int n_groups;
    int64_t n_tasks;
    int phases, run_rows;
    float* S;
};

// KH k-steps of 32 coordinates are one unit of the walk: what is prefetched and what is unrolled.  A gallery block
// is `phases` units; up to 192 coordinates it is one.
template <int KH, int TT>  // TT: tiles of 16 tests
__global__ __launch_bounds__(256, TT == 4 ? 2 : 3) void q4_score_kernel(Q4Args g) {
#if defined(__HIP_DEVICE_COMPILE__)
    extern __shared__ __attribute__((aligned(16))) uint4 test[];  // [TT][ks][2][64]
    __shared__ __attribute__((aligned(16))) int up_s[16 * TT];
    __shared__ __attribute__((aligned(16))) float add_s[16 * TT];

    const int64_t t = xcd_task(blockIdx.x, g.n_tasks, Q4_RUN);
    if (t < 0) return;
    const int e = find_group(g.tasks, g.n_groups, t);
    const int64_t n = g.off_g[e + 1] - g.off_g[e], m_all = g.off_t[e + 1] - g.off_t[e];
    const int64_t runs = (n + g.run_rows - 1) / g.run_rows;
    const int64_t task = t - g.tasks[e];
    const int64_t tb = task / runs, run = task - tb * runs;
    const int64_t t0 = tb * 16 * TT;
    const int m = m_all - t0 < 16 * TT ? (int)(m_all - t0) : 16 * TT;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kq = lane >> 4;
    const int ks_all = KH * g.phases;

    // ---- gallery blocks of this wave: wave, wave + 4, ... of the run
    const int64_t row0 = run * g.run_rows;
    const int nb = (int)(((n - row0 < g.run_rows ? n - row0 : g.run_rows) + Q4_BLOCK - 1) / Q4_BLOCK);
    const int64_t b0 = g.blk[e] + row0 / Q4_BLOCK;
    const int units = wave < nb ? ((nb - wave + 3) >> 2) * g.phases : 0;
    uint4 c[KH];
    uint2 s[KH];
    float qv[4] = {0.f, 0.f, 0.f, 0.f};
    int b_next = wave, ph_next = 0;
    auto fetch = [&]() {
        const int64_t at = (b0 + b_next) * ks_all + ph_next * KH;
        const uint4* pc = g.codes + at * 64 + lane;
        const uint2* ps = g.scales + at * 16 + r16;
#pragma unroll
        for (int ks = 0; ks < KH; ++ks) {
            c[ks] = pc[ks * 64];
            s[ks] = ps[ks * 16];
        }
        if (++ph_next == g.phases) {
            const float* pq = g.q + (b0 + b_next) * Q4_BLOCK + r16;
#pragma unroll
            for (int u = 0; u < 4; ++u) qv[u] = pq[16 * u];
            ph_next = 0;
            b_next += 4;
        }
    };
    if (units) fetch();

    // ---- tests: lane holds coordinates 32 ks + 8 kq .. + 7 of test r16 of a tile.  4 / TT waves share a tile: each
    // reads all of it (one latency, whatever its width) and prepares every (4 / TT)th k-step.
    {
        const int tt = wave % TT, ti = 16 * tt + r16;
        const float* p = g.G + (g.off_t[e] + t0 + (ti < m ? ti : 0)) * g.ld;
        float top = 0.f;
        auto coords = [&](int ks, f32x4& lo, f32x4& hi) {
            const int k = 32 * ks + 8 * kq, at = k < g.k ? k : (g.k - 1) & ~7;
            lo = *reinterpret_cast<const f32x4*>(p + at);
            hi = *reinterpret_cast<const f32x4*>(p + at + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // q and the padding of a row lie behind its coordinates
                lo[j] = (ti < m && k + j < g.k) ? lo[j] : 0.f;
                hi[j] = (ti < m && k + 4 + j < g.k) ? hi[j] : 0.f;
            }
        };
#pragma unroll 4
        for (int ks = 0; ks < ks_all; ++ks) {
            f32x4 lo, hi;
            coords(ks, lo, hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(fabsf(lo[j]), fabsf(hi[j])));
        }
        top = swap32_max(swap16_max(top));
        int up = top > 0.f ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
        up = up > 126 ? 126 : up;
        const float f = exp2_int(up);
        for (int ks = wave / TT; ks < ks_all; ks += 4 / TT) {
            f32x4 lo, hi;
            coords(ks, lo, hi);
            f16x4 l0, l1, h0, h1;
            split_pair4(lo, f, l0, l1);
            split_pair4(hi, f, h0, h1);
            uint4* dst = &test[((tt * ks_all + ks) * 2) * 64 + lane];
            dst[0] = __builtin_bit_cast(uint4, __builtin_shufflevector(l0, h0, 0, 1, 2, 3, 4, 5, 6, 7));
            dst[64] = __builtin_bit_cast(uint4, __builtin_shufflevector(l1, h1, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        if (wave < TT && kq == 0) {
            up_s[ti] = -up;
            add_s[ti] = ti < m ? p[g.k + 1] : 0.f;
        }
    }
    __syncthreads();

    const f16x2 lo8 = {(_Float16)-1032.f, (_Float16)-1032.f}, hi8 = {(_Float16)-72.f, (_Float16)-72.f};
    const f16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const unsigned exponent = 0x64006400u;  // 1024 twice
    auto nibbles = [&](unsigned w, unsigned mask) {  // (w & mask) | exponent, in one instruction
        unsigned r;
        asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(exponent));
        return __builtin_bit_cast(f16x2, r);
    };

    float* out = g.S + g.out[e] + t0 * n + row0;
    f32x4 acc[TT][4];
    int b = wave, ph = 0;
    for (int it = 0; it < units; ++it) {
        asm volatile("" ::: "memory");  // the test operands stay in LDS: hoisted, they are the registers of two waves
        if (ph == 0) {
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[tt][u] = (f32x4){0.f, 0.f, 0.f, 0.f};
        }
        float qb[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) qb[u] = qv[u];
        uint4 cc[KH];
        uint2 sc[KH];
#pragma unroll
        for (int ks = 0; ks < KH; ++ks) {
            cc[ks] = c[ks];
            sc[ks] = s[ks];
        }
        if (it + 1 < units) fetch();
#pragma unroll
        for (int ks = 0; ks < KH; ++ks) {
            const unsigned w[4] = {cc[ks].x, cc[ks].y, cc[ks].z, cc[ks].w};
            f16x8 op[4];
            float sf[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const unsigned h = w[u] >> 8;
                f16x2 o[4];
                o[0] = nibbles(w[u], 0x000f000fu) + lo8;
                o[1] = __builtin_elementwise_fma(nibbles(w[u], 0x00f000f0u), sixteenth, hi8);
                o[2] = nibbles(h, 0x000f000fu) + lo8;
                o[3] = __builtin_elementwise_fma(nibbles(h, 0x00f000f0u), sixteenth, hi8);
                op[u] = __builtin_bit_cast(f16x8, o);
                const unsigned p = u < 2 ? sc[ks].x : sc[ks].y;
                sf[u] = __uint_as_float((u & 1) ? p & 0xffff0000u : p << 16);
            }
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const int at = tt * ks_all + ph * KH + ks;
                const f32x4 c0 = {0.f, 0.f, 0.f, 0.f};
                const f16x8 a0 = __builtin_bit_cast(f16x8, test[at * 128 + lane]);
                const f16x8 a1 = __builtin_bit_cast(f16x8, test[at * 128 + 64 + lane]);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    f32x4 d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, op[u], c0, 0, 0, 0);
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, op[u], d, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[tt][u][r] = fmaf(sf[u], d[r], acc[tt][u][r]);
                }
            }
        }
        if (++ph < g.phases) continue;
        ph = 0;
        // lane: tests 16 tt + 4 kq + r, gallery rows 64 b + 16 u + r16
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int4 up = *reinterpret_cast<const int4*>(&up_s[16 * tt + 4 * kq]);
            const f32x4 add = *reinterpret_cast<const f32x4*>(&add_s[16 * tt + 4 * kq]);
            const int upv[4] = {up.x, up.y, up.z, up.w};
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int ti = 16 * tt + 4 * kq + r;
                if (ti >= m) continue;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int64_t row = (int64_t)b * Q4_BLOCK + 16 * u + r16;
                    if (row0 + row < n) out[ti * n + row] = (ldexpf(acc[tt][u][r], upv[r]) + qb[u]) + add[r];
                }
            }
        }
        b += 4;
    }
#endif
}

template <int KH, int TT>
int launch_q4(const Q4Args& g, hipStream_t stream) {
    const int64_t grid = xcd_grid(g.n_tasks, Q4_RUN);
    HYPMI_REQUIRE(fits_launch(grid, 256), "q4_score: too many workgroups");
    const int lds = TT * KH * g.phases * 2048;
    if (lds > 48 * 1024)
        HYPMI_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&q4_score_kernel<KH, TT>),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    hipLaunchKernelGGL((q4_score_kernel<KH, TT>), dim3((unsigned)grid), dim3(256), lds, stream, g);
    HYPMI_HIP(hipGetLastError());
    return HYPMI_OK;
}

template <int KH>
int launch_q4_tests(const Q4Args& g, int tests, hipStream_t stream) {
    switch (tests) {
        case 16: return launch_q4<KH, 1>(g, stream);
        case 32: return launch_q4<KH, 2>(g, stream);
        default: return launch_q4<KH, 4>(g, stream);
    }
}

constexpr int Q4_MAX_KS = 16;

}  // namespace hypmi_detail

using namespace hypmi_detail;

static int q4_ksteps(int k) {
    const int ks = (k + 31) / 32;
    return (k <= 0 || ks > Q4_MAX_KS) ? 0 : ks <= 6 ? ks : ks <= 8 ? 8 : ks <= 10 ? 10 : ks <= 12 ? 12 : 16;
}

extern "C" int hypmi_q4_ksteps(int k) { return q4_ksteps(k); }

extern "C" int hypmi_q4_rows(const float* G, int64_t ldg, int k, const int64_t* offsets, const int64_t* blocks,
                             int n_groups, int64_t n_blocks, void* codes, void* scales, float* q, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    const int ks = q4_ksteps(k);
    HYPMI_REQUIRE(ks > 0, "q4_rows: %d coordinates (1 to 512)", k);
    HYPMI_REQUIRE(fits_groups(n_groups) && n_blocks >= 0 && ldg >= k + 1, "q4_rows: bad shape");
    if (n_blocks == 0) return HYPMI_OK;
    HYPMI_REQUIRE(G && offsets && blocks && codes && scales && q, "q4_rows: null pointer");
    HYPMI_REQUIRE(aligned16(codes) && aligned16(scales), "q4_rows: buffers must be 16-byte aligned");
    const int64_t grid = (n_blocks * ks + 3) / 4;
    HYPMI_REQUIRE(fits_launch(grid, 256), "q4_rows: too many rows");
    hipLaunchKernelGGL(q4_rows_kernel, dim3((unsigned)grid), dim3(256), 0, stream, G, ldg, k, ks, offsets, blocks,
                       n_groups, n_blocks, static_cast<unsigned*>(codes), static_cast<unsigned short*>(scales), q);
    HYPMI_HIP(hipGetLastError());
    return HYPMI_OK;
}

extern "C" int hypmi_q4_score(const void* codes, const void* scales, const float* q, int k, const float* G, int64_t ldg,
                              const int64_t* offsets_t, const int64_t* offsets_g, const int64_t* blocks,
                              const int64_t* out_offsets, const int64_t* tasks, int task_tests, int task_rows,
                              int n_groups, int64_t n_tasks, float* S, void* stream_) {
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    const int ks = q4_ksteps(k);
    HYPMI_REQUIRE(ks > 0, "q4_score: %d coordinates (1 to 512)", k);
    HYPMI_REQUIRE(task_tests == 16 || task_tests == 32 || task_tests == 64, "q4_score: 16, 32 or 64 tests per task");
    HYPMI_REQUIRE(task_rows > 0 && task_rows % Q4_BLOCK == 0, "q4_score: task_rows must be a multiple of 64");
    HYPMI_REQUIRE(fits_groups(n_groups) && n_tasks >= 0, "q4_score: bad shape");
    HYPMI_REQUIRE(ldg % 4 == 0 && ldg >= k + 2 && ldg >= (k + 7) / 8 * 8, "q4_score: bad leading dimension");
    if (n_tasks == 0) return HYPMI_OK;
    HYPMI_REQUIRE(codes && scales && q && G && offsets_t && offsets_g && blocks && out_offsets && tasks && S,
                  "q4_score: null pointer");
    HYPMI_REQUIRE(aligned16(codes) && aligned16(scales) && aligned16(G), "q4_score: buffers must be 16-byte aligned");
    const int phases = ks <= 6 ? 1 : ks == 16 ? 4 : 2;
    const Q4Args g = {static_cast<const uint4*>(codes), static_cast<const uint2*>(scales), q, G, ldg, k, offsets_t,
                      offsets_g, blocks, out_offsets, tasks, n_groups, n_tasks, phases, task_rows, S};
    switch (ks / phases) {
        case 1: return launch_q4_tests<1>(g, task_tests, stream);
        case 2: return launch_q4_tests<2>(g, task_tests, stream);
        case 3: return launch_q4_tests<3>(g, task_tests, stream);
        case 4: return launch_q4_tests<4>(g, task_tests, stream);
        case 5: return launch_q4_tests<5>(g, task_tests, stream);
        default: return launch_q4_tests<6>(g, task_tests, stream);
    }
}
