// What the attentions over a cache of 4 bits an element share: queries in two 8-bit parts, and the merge of partial results.
#pragma once

#include "four_bit.h"

#include <math.h>

namespace leone {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4;
typedef int intx8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.0f;                     // a score this far above the reference raises it

__device__ inline intx8 low_half(uint4 v) { return intx8{static_cast<int>(v.x), static_cast<int>(v.y), static_cast<int>(v.z), static_cast<int>(v.w), 0, 0, 0, 0}; }

// A query row as two 8-bit parts: sixteen elements a call, `unit` 2^-e with the row's largest element in [2^7, 2^8) units.  The rest is
// at most half of the first part's last place, which is sixteen units at most: times 32 it is no larger than 2^8.
__device__ inline void two_parts(const uint4 raw[2], float unit, int high[4], int low[4]) {
    const unsigned w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x[4];
        x[0] = __uint_as_float(w[2 * i] << 16) * unit, x[1] = __uint_as_float(w[2 * i] & 0xffff0000u) * unit;
        x[2] = __uint_as_float(w[2 * i + 1] << 16) * unit, x[3] = __uint_as_float(w[2 * i + 1] & 0xffff0000u) * unit;
        int h = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        h = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], h, true);
        const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8(h, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(h, true);
        int r = __builtin_amdgcn_cvt_pk_fp8_f32((x[0] - a[0]) * 32.f, (x[1] - a[1]) * 32.f, 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32((x[2] - b[0]) * 32.f, (x[3] - b[1]) * 32.f, r, true);
        high[i] = h, low[i] = r;
    }
}
__device__ inline unsigned largest_bits(uint4 v, unsigned top) {          // of eight bfloat16, as the bits of a float
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(max(top, w[i] & 0x7fff0000u), w[i] << 16 & 0x7fff0000u);
    return top;
}
// The power byte of a row's first part, from its largest element's bits: 255 where it is no number (its scores are then NaN).  It is at
// least 6, so that the rest's is at least 1: rows of nothing larger than 2^-114 keep fewer bits.
__device__ inline int query_power(unsigned top) {
    const int exponent = static_cast<int>(top >> 23);
    return exponent == 0xff ? kNanPower : max(exponent - 7, 6);
}
__device__ inline float query_unit(int power) { return __uint_as_float(static_cast<unsigned>(254 - (power == kNanPower ? 127 : power)) << 23); }
__device__ inline int rest_power(int power) { return power == kNanPower ? kNanPower : power - 5; }

inline FourBitPools read_pools(const void* k_codes, const void* k_powers, const void* v_codes, const void* v_powers, int pages) {
    auto bytes = [](const void* p) { return const_cast<uint8_t*>(static_cast<const uint8_t*>(p)); };
    return FourBitPools{bytes(k_codes), bytes(k_powers), bytes(v_codes), bytes(v_powers), pages};
}


// Merges the shares of a (row, query head) in their order: sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M), from part_acc [rows *
// q_heads, splits, dim] and part_ml [rows * q_heads, splits, 2]; shares with a maximum of -inf count as nothing, a row with no other
// gives zeros.  With a list of tiles (entry, first row, rows up to 32) `rows` is their number times 32 and the rows are theirs, as far as
// they lie below `limit`.
constexpr int kShares = kWave;                     // the most shares
constexpr int kTileRows = 32;
void merge_four_bit_shares(const float* part_acc, const float* part_ml, void* out, int dtype, long rows, int q_heads, int dim, int splits,
                           const int* tiles, int limit, hipStream_t stream);

}  // namespace leone
