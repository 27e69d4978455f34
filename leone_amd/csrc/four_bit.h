// The cache of 4 bits an element: blocks of 32 consecutive elements of a token's key or value vector, each a number of the
// 4-bit floating type e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) times the block's own power of two, 2^(byte - 127)
// (MXFP4 of the Open Compute Project's Microscaling specification, which this chip's matrix instructions and conversions
// take as it is).  The power is the smallest whose sevenfold is not below the block's largest magnitude: numbers up to 7
// round to 6, so that nothing is off by more than one unit, the most that is lost between 4 and 6 as well.  A block with a NaN or an
// infinity in it gets byte 255 and stands for NaN.  (Numbers from 1.75 x 2^127 up round to 2^128 or more, which is an infinity as a
// bfloat16 or a float.)
//
// Layout, P tokens a page:
//   key codes     [page][kv head][dim / 32][P][16 bytes]          a block: what a lane of the first product takes
//   key powers    [page][kv head][P][dim / 32]                    a token's, side by side
//   value codes   [page][kv head][P / 4][dim / 8][4 tokens][4 bytes]  eight neighbouring elements of four tokens: the second
//                                                                 product sums over tokens, a lane needs several of an element
//   value powers  [page][kv head][P / 4][dim / 32][4 tokens]
// Two codes a byte, the lower element in the low half.
#pragma once

#include "common.h"

namespace leone {

constexpr int kBlock = 32;                         // elements that share a power of two
constexpr int kNanPower = 255;
// Tokens that a block table may reach, and the last position that is told from those behind it (all of them without a page): what is
// computed from positions stays within 32 bits.
constexpr int kReach = 1 << 30;
constexpr int kLastPosition = kReach + (1 << 20);

struct FourBitPools {
    uint8_t* k_codes;
    uint8_t* k_powers;
    uint8_t* v_codes;
    uint8_t* v_powers;
    int pages;
};

// One page of one kv head, in bytes.
__host__ __device__ inline long four_bit_codes(int page_tokens, int dim) { return static_cast<long>(page_tokens) * dim / 2; }
__host__ __device__ inline long four_bit_powers(int page_tokens, int dim) { return static_cast<long>(page_tokens) * (dim / kBlock); }

// Where things lie within a page of one kv head.
__host__ __device__ inline int four_bit_key(int token, int block, int page_tokens) { return (block * page_tokens + token) * 16; }
__host__ __device__ inline int four_bit_key_power(int token, int block, int dim) { return token * (dim / kBlock) + block; }
__host__ __device__ inline int four_bit_value(int token, int eight, int dim) { return ((token >> 2) * (dim / 8) + eight) * 16 + (token & 3) * 4; }
__host__ __device__ inline int four_bit_value_power(int token, int block, int dim) { return ((token >> 2) * (dim / kBlock) + block) * 4 + (token & 3); }

// 2^(byte - 127) as the conversions take it: they read the exponent alone, and one of 255 gives NaN.
__device__ inline float power_of(unsigned byte) { return __uint_as_float(byte << 23); }

// Codes 2 i and 2 i + 1 of a word of eight, as the numbers they stand for.
typedef float floatx2 __attribute__((ext_vector_type(2)));
template <int i>
__device__ inline floatx2 two_floats(unsigned codes, float power) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, power, i);
}
template <int i>
__device__ inline unsigned two_bf16(unsigned codes, float power) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, power, i));
}
__device__ inline void eight_floats(unsigned codes, float power, float out[8]) {
    const floatx2 a = two_floats<0>(codes, power), b = two_floats<1>(codes, power), c = two_floats<2>(codes, power), d = two_floats<3>(codes, power);
    out[0] = a[0], out[1] = a[1], out[2] = b[0], out[3] = b[1], out[4] = c[0], out[5] = c[1], out[6] = d[0], out[7] = d[1];
}

// The page of a request's position, -1 where it has none: a position behind the table, or a table entry that is no page.
__device__ inline int mapped_page(const int* __restrict__ table, int block, int max_blocks, int pages) {
    if (block >= max_blocks) return -1;
    const int page = table[block];
    return page < pages ? page : -1;
}

inline int check_four_bit(const char* what, const FourBitPools& p, int kv_heads, int dim, int page_tokens, int max_blocks) {
    LEONE_REQUIRE(p.k_codes && p.k_powers && p.v_codes && p.v_powers, "%s: null pool", what);
    LEONE_REQUIRE((reinterpret_cast<uintptr_t>(p.k_codes) | reinterpret_cast<uintptr_t>(p.k_powers) | reinterpret_cast<uintptr_t>(p.v_codes) |
                   reinterpret_cast<uintptr_t>(p.v_powers)) % 16 == 0, "%s: the pools start at multiples of 16 bytes", what);
    LEONE_REQUIRE(p.pages > 0 && kv_heads > 0 && max_blocks > 0, "%s: %d pages, %d kv heads, block tables of %d", what, p.pages, kv_heads, max_blocks);
    LEONE_REQUIRE(static_cast<long>(max_blocks) * page_tokens <= kReach, "%s: block tables of %d pages of %d tokens reach further than 2^30 tokens", what,
                  max_blocks, page_tokens);
    LEONE_REQUIRE(dim % kBlock == 0 && dim >= kBlock && dim <= 256, "%s: heads of %d elements; blocks of 32 need a multiple of 32 up to 256", what, dim);
    LEONE_REQUIRE(page_tokens % 8 == 0 && page_tokens >= 8 && page_tokens <= 4096, "%s: pages of %d tokens; a multiple of 8 up to 4,096 is needed", what, page_tokens);
    return 0;
}

}  // namespace leone
