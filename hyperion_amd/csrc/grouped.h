// Shared device code of the grouped operators (grouped_affine.hip, grouped_score.hip, grouped_gram.hip,
// gallery.hip): rows that fall into groups of unequal sizes, delimited by offsets, are cut into tiles that
// never cross a group; a workgroup finds its (group, tile) from a prefix sum of the tile counts.
#pragma once
#include "common.h"

namespace hypmi_detail {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
// rows of caller arrays start at any multiple of their element size
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// Largest e with prefix[e] <= t, for prefix[0] = 0 <= t < prefix[n]: the group of tile t (groups without
// tiles share their successor's entry and are never returned).  All 64 lanes of a wave probe at once, so a
// thousand groups take two dependent loads.  Call it with the whole wave active.
__device__ __forceinline__ int find_group(const int64_t* __restrict__ prefix, int n, int64_t t) {
    const int lane = (int)(threadIdx.x & 63);
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) >> 6;
        const int64_t p = lo + (int64_t)(lane + 1) * step;
        const bool le = p < hi && prefix[p] <= t;
        const int c = __popcll(__ballot(le));
        lo += c * step;
        hi = lo + step < hi ? lo + step : hi;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// Workgroups are handed to the eight XCDs round robin (a placement assumed for speed only).  Runs of `run` tasks are
// dealt to the XCDs in turn: neighbouring tasks, which read the same operands, meet in one L2, and tasks of unequal
// cost, which also stand together, do not end up on one XCD.  Returns -1 for the slots that pad the grid.
__device__ __forceinline__ int64_t xcd_task(int64_t b, int64_t n, int run) {
    const int64_t k = b >> 3, t = ((k / run) * 8 + (b & 7)) * run + k % run;
    return t < n ? t : -1;
}

// What find_group counts in 32 bits: the number of groups, and that and a step more.
inline bool fits_groups(int n) { return n >= 0 && n <= 1 << 30; }

// A launch holds fewer than 2^32 work-items in a dimension.
inline bool fits_launch(int64_t blocks, int threads) { return blocks >= 0 && blocks <= 0xffffffffLL / threads; }

inline int64_t xcd_grid(int64_t n, int run) { return (n + 8 * run - 1) / (8 * run) * (8 * run); }

// 2^e as a float, -126 <= e <= 127
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// x up -> x0 + x1 with x0 = fp16(x up), x1 = fp16(x up - x0), four values and a power of two `up`:
// |x up - x0 - x1| <= 2^-22 |x up| while x1 is a normal fp16 number.  An infinity becomes (inf, NaN): its products
// are NaN.  Three instructions a value (v_mul, half a v_cvt_pk_f16_f32, v_fma_mix_f32, half a v_cvt_pk_f16_f32).
__device__ __forceinline__ void split_pair4(f32x4 x, float up, f16x4& x0, f16x4& x1) {
    x0 = __builtin_convertvector(x * up, f16x4);
    f32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = fmaf(x[i], up, -(float)x0[i]);
    x1 = __builtin_convertvector(r, f16x4);
}

// max(x, x of another lane) by a data-parallel-primitive control: 0xB1 lane ^ 1, 0x4E lane ^ 2, 0x141 the mirror
// image within eight lanes, 0x140 within sixteen
template <int CTRL>
__device__ __forceinline__ float dpp_max(float x) {
    const int y = __builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true);
    return fmaxf(x, __int_as_float(y));
}

// max over the lanes l ^ 16, over l ^ 32 (vector instructions; a shuffle goes through LDS)
__device__ __forceinline__ float swap16_max(float x) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float swap32_max(float x) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

}  // namespace hypmi_detail
