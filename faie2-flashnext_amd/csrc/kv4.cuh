// The 4-bit paged cache: format, page layout, and rows in and out of it.
//
// A value is an e2m1 code (sign, magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) times 2^(s - 127), one scale byte s for 32 dims of
// a row.  This is the block format that the matrix cores of gfx950 take as an operand, so K is never converted; V is
// converted by one instruction for two values and its values are exact in bf16.
// A page holds 64 tokens of every key/value head, HEAD_BYTES a head: K codes, K scales, V codes, V scales.
//   K codes  [64-token 16-key block 4][half of the row 2][group of the half 4][key 16][16 bytes: 32 dims, low nibble
//            first]: a wave's A operand of v_mfma_scale_f32_16x16x128_f8f6f4 is 1 KiB in a row, 16 bytes a lane.
//   K scales [32-key block 2][group of the half 4][key 16][16-key block 2][half of the row 2]: the four scales of a lane's
//            operands in 32 keys are one dword, and the instruction picks the byte.
//   V codes  [32-key block 2][pair of groups 4][quarter 4][pair of dims 16][group of the pair 2][key 8]: a byte is dims
//            2m, 2m + 1 of one key; quarter q holds keys 4q .. 4q + 3 of the first and of the second 16-key block, the
//            keys whose probabilities the scores' layout leaves in the lanes of quarter q.
//   V scales [32-key block 2][quarter 4][group 8][key 8].
#pragma once

#include "serve.h"

namespace fn {

namespace kv4 {

constexpr int HD = 256, PG = 64;                 // head dim built, tokens a page
constexpr int CODES = PG * HD / 2, SCALES = PG * HD / 32;
constexpr int KS = CODES, VC = CODES + SCALES, VS = 2 * CODES + SCALES;
constexpr int HEAD_BYTES = 2 * (CODES + SCALES);  // 17408
// The scale of a group is the least power of two that leaves its largest value off by at most half a step, kept
// between these: what a lower one would hold is below 2^-101, and with the upper one every code is finite in fp32.
constexpr int EMIN = -100, EMAX = 125;

// byte offset in a head's page of: the 16 bytes of K group grp of row r; its scale; V's byte of dims 32 grp + 2m, + 1; scale
__device__ __forceinline__ int k_code(int r, int grp) {
    return (((r / 16 * 2 + grp / 4) * 4 + grp % 4) * 16 + r % 16) * 16;
}
__device__ __forceinline__ int k_scale(int r, int grp) {
    return KS + ((r / 32 * 4 + grp % 4) * 16 + r % 16) * 4 + r % 32 / 16 * 2 + grp / 4;
}
__device__ __forceinline__ int v_code(int r, int grp, int m) {
    return VC + ((r / 32 * 4 + grp / 2) * 64 + r % 16 / 4 * 16 + m) * 16 + grp % 2 * 8 + r % 32 / 16 * 4 + r % 4;
}
__device__ __forceinline__ int v_scale(int r, int grp) {
    return VS + ((r / 32 * 4 + r % 16 / 4) * 8 + grp) * 8 + r % 32 / 16 * 4 + r % 4;
}

// Code of |u| in scale units: nearest, ties to the even code.
__device__ __forceinline__ uint32_t code_of(double u) {
    return (u > 0.25) + (u >= 0.75) + (u > 1.25) + (u >= 1.75) + (u > 2.5) + (u >= 3.5) + (u > 5.0);
}

// One row of HD values by a wave, lane = dims 4l .. 4l + 3, into row r of a head's page as K or as V.  The values are
// in float64: a code is the nearest to the exact value, and a key's norm and rotation in fp32 would move values across
// the borders between codes.  A group with an infinity or NaN has no 4-bit form: it is stored as zeros and the status
// word says so.
template <bool IS_K>
__device__ __forceinline__ void store_row(uint8_t *page, int r, const double (&y)[4], int lane, unsigned *status) {
    double a = 0.0;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bad |= !(fabs(y[i]) < INFINITY);
        a = fmax(a, fabs(y[i]));
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) {
        a = fmax(a, __shfl_xor(a, d));
        bad |= __shfl_xor((int) bad, d) != 0;
    }
    int e = EMIN;
    if (!bad && a > 0.0) {
        const uint64_t w = __builtin_bit_cast(uint64_t, a);
        e = (int) ((w >> 52) & 0x7ff) - 1023 - 2;                // a in [4, 8) 2^e
        e += (w & 0xFFFFFFFFFFFFFull) > 0xC000000000000ull;     // above 7: the next scale
        e = max(EMIN, min(EMAX, e));
    }
    uint32_t c = 0;
    if (!bad) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c |= (code_of(ldexp(fabs(y[i]), -e)) | (__builtin_bit_cast(uint64_t, y[i]) >> 63) << 3) << (4 * i);
    } else if ((lane & 7) == 0) {
        atomicOr(status, FN_STATUS_VALUE);
    }
    const int grp = lane >> 3, sub = lane & 7;
    if (IS_K) {
        *reinterpret_cast<uint16_t *>(page + k_code(r, grp) + sub * 2) = (uint16_t) c;
        if (sub == 0) page[k_scale(r, grp)] = (uint8_t) (e + 127);
    } else {
        page[v_code(r, grp, 2 * sub)] = (uint8_t) c;
        page[v_code(r, grp, 2 * sub + 1)] = (uint8_t) (c >> 8);
        if (sub == 0) page[v_scale(r, grp)] = (uint8_t) (e + 127);
    }
}

__device__ __forceinline__ float value_of(uint32_t code, int s) {
    const uint32_t m = code & 7;
    const float x = m < 2 ? 0.5f * m : (float) (2 + (m & 1)) * (float) (1 << (m >> 1)) * 0.25f;
    return ldexpf(code & 8 ? -x : x, s - 127);
}

}  // namespace kv4

}  // namespace fn
