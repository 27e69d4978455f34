// Attention of single rows over the cache of 4 bits an element (four_bit.h): one kernel for every shape and type, one
// for single tokens on the matrix cores, and the merge of both's partial results.
//
// A row at position p sees the keys [first_key(p, window), p] of its request; a row that sees none (position -1) gives
// zeros; a key in sight whose place has no page makes the row's result NaN.  All softmax statistics and sums are float, in powers of two
// (score * scale * log2(e)).
//
// ---- single tokens (decode), bfloat16, heads of 64, 128 and 256 -------------------------------------------------------
// A workgroup takes (row, kv head, up to 16 of its query heads, one share of the keys); its four waves walk 32-key tiles of the
// share.  What it waits for is the cache, a 3.8th of a bfloat16 one, so the work an element costs is what counts:
// a compute unit gets some 23 elements a cycle from memory and has 64 lanes' instructions a cycle.  So
//  * the first product takes the keys as they lie in the cache, v_mfma_scale_f32_16x16x128_f8f6f4 with 4-bit keys and their powers and
//    8-bit queries, and nothing is unpacked.  A query is two 8-bit numbers (e4m3, one power of two a row): its four leading bits
//    and, by a second product, the rest.  The eight bits of a bfloat16 are kept whole down to 2^-21 of the row's largest element.
//    Heads of 64 hold both parts in one product, the keys given twice.
//  * the values are unpacked by the chip's own conversion, two to an instruction with their power, and brought from neighbouring
//    elements of a token to neighbouring tokens of an element by one byte permutation for two.  The second product is then
//    v_mfma_f32_16x16x32_bf16 on exact values; its weights are rounded to bfloat16, against a reference that is a whole number, so
//    that the rounding does not depend on how the keys are cut, and the sum is taken over the rounded weights.
// Operand layouts (lane l, c = l % 16, g = l / 16), checked on the chip: 4-bit operand: row c, elements 32 g .. + 31; 8-bit operand:
// column c, elements 16 g .. + 15 and 64 + 16 g .. + 15; a lane's power belongs to elements 32 g .. + 31 of its row or column.
// Result: column c, rows 4 g .. + 3.  Row c of the first half of a tile is key 8 (c / 4) + c % 4, of the second four further, so
// that a lane's scores are those of keys 8 g .. + 7 and go into the second product as they are.
// The reference is raised only by a score that exceeds it by more than 8 (weights stay below 2^8): no exchange between lanes
// otherwise.
#include "common.h"
#include "four_bit.h"
#include "leone_hip.h"
#include "score_shape.h"

#include <math.h>

namespace leone {

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4;
typedef int intx8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;

// ---- any shape and type ------------------------------------------------------------------------------------------------
// A workgroup takes (row, kv head, up to four of its query heads, one share of the keys), a wave 64 keys at a time: a lane takes a
// key for the scores, and eight elements of every kSubs-th run of four tokens for the results.
constexpr int kRowsWaves = 4;
constexpr int kRowsThreads = kRowsWaves * kWave;
constexpr int kRowsHeads = 4;
constexpr int kRowsKeys = kWave;

template <int kBlocks, typename T>
__global__ void __launch_bounds__(kRowsThreads)
four_bit_attend_rows_kernel(const T* __restrict__ q, T* __restrict__ out, FourBitPools pools, const int* __restrict__ positions,
                            const int* __restrict__ row_entry, const int* __restrict__ block_table, int max_blocks, int entries, int q_heads,
                            int kv_heads, int page_tokens, float to_log2, int window, int splits, float* __restrict__ part_acc,
                            float* __restrict__ part_ml) {
    constexpr int kD = kBlocks * kBlock, kEights = kD / 8;
    constexpr int kSubs = kWave / kEights;                       // lanes behind kSubs * kEights have no values to add up
    __shared__ float4 q_held[kRowsHeads][kD / 4];
    __shared__ float weight[kRowsWaves][kRowsHeads][kRowsKeys];
    __shared__ int page_held[kRowsWaves][kRowsKeys];
    __shared__ float part[kRowsWaves][kRowsHeads][kD];
    __shared__ float part_m[kRowsWaves][kRowsHeads], part_l[kRowsWaves][kRowsHeads];
    const int group = q_heads / kv_heads, head_tiles = (group + kRowsHeads - 1) / kRowsHeads;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int row = blockIdx.x, kvh = blockIdx.y / head_tiles, head0 = kvh * group + blockIdx.y % head_tiles * kRowsHeads;
    const int heads = min(kRowsHeads, (kvh + 1) * group - head0);
    const int entry = row_entry[row];
    const int n = entry >= 0 && entry < entries ? positions[row] + 1 : 0;
    const int lo = first_key(n - 1, window, 0);
    const int* table = block_table + static_cast<long>(entry) * max_blocks;
    for (int i = threadIdx.x; i < kRowsHeads * kD; i += kRowsThreads) {
        const int h = i / kD, d = i % kD;
        reinterpret_cast<float*>(q_held)[i] = h < heads ? to_float(q[(static_cast<long>(row) * q_heads + head0 + h) * kD + d]) : 0.f;
    }
    __syncthreads();
    float acc[kRowsHeads][8], m[kRowsHeads], l[kRowsHeads];
#pragma unroll
    for (int h = 0; h < kRowsHeads; ++h) {
        m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[h][i] = 0.f;
    }
    bool unmapped = false;
    const int t_begin = lo / kRowsKeys, t_end = (n + kRowsKeys - 1) / kRowsKeys;
    const int share = (t_end - t_begin + splits - 1) / splits;
    const int my_begin = t_begin + static_cast<int>(blockIdx.z) * share, my_end = min(my_begin + share, t_end);
    const int eight = lane % kEights, sub = lane / kEights;
    for (int t = my_begin + wave; t < my_end; t += kRowsWaves) {
        const int key = t * kRowsKeys + lane;
        const bool seen = key >= lo && key < n;
        const int page = seen ? mapped_page(table, key / page_tokens, max_blocks, pools.pages) : -1;
        const int token = key % page_tokens;
        unmapped |= seen && page < 0;
        float score[kRowsHeads] = {0.f, 0.f, 0.f, 0.f};
        if (page >= 0) {
            const long place = static_cast<long>(page) * kv_heads + kvh;
            const uint8_t* codes = pools.k_codes + place * four_bit_codes(page_tokens, kD);
            const uint8_t* powers = pools.k_powers + place * four_bit_powers(page_tokens, kD) + four_bit_key_power(token, 0, kD);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const uint4 raw = *reinterpret_cast<const uint4*>(codes + four_bit_key(token, b, page_tokens));
                const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
                const float power = power_of(powers[b]);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    float x[8];
                    eight_floats(words[w], power, x);
#pragma unroll
                    for (int h = 0; h < kRowsHeads; ++h) {
                        const float4 a = q_held[h][b * 8 + w * 2], c = q_held[h][b * 8 + w * 2 + 1];
                        score[h] = fmaf(x[0], a.x, fmaf(x[1], a.y, fmaf(x[2], a.z, fmaf(x[3], a.w, score[h]))));
                        score[h] = fmaf(x[4], c.x, fmaf(x[5], c.y, fmaf(x[6], c.z, fmaf(x[7], c.w, score[h]))));
                    }
                }
            }
        }
        page_held[wave][lane] = page;
#pragma unroll
        for (int h = 0; h < kRowsHeads; ++h) {
            const float s = page >= 0 ? score[h] * to_log2 : -INFINITY;
            const float top = fmaxf(m[h], wave_max(s));
            const float p = top == -INFINITY ? (s == s ? 0.f : s) : __builtin_amdgcn_exp2f(s - top);
            const float keep = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[h] - top);
            l[h] = l[h] * keep + wave_sum(p);
            m[h] = top;
            weight[wave][h][lane] = p;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[h][i] *= keep;
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // this wave's own writes; no other reads them
        if (sub < kSubs) {
            for (int run = sub; run < kRowsKeys / 4; run += kSubs) {
                int key4 = t * kRowsKeys + 4 * run;
                int page4 = -1;                                   // (a run may begin before the first key in sight)
#pragma unroll
                for (int i = 0; i < 4; ++i) page4 = max(page4, page_held[wave][4 * run + i]);
                if (page4 < 0) continue;
                const int token4 = key4 % page_tokens;
                const long place = static_cast<long>(page4) * kv_heads + kvh;
                const uint4 raw = *reinterpret_cast<const uint4*>(pools.v_codes + place * four_bit_codes(page_tokens, kD) + four_bit_value(token4, eight, kD));
                const unsigned powers = *reinterpret_cast<const unsigned*>(pools.v_powers + place * four_bit_powers(page_tokens, kD) +
                                                                           four_bit_value_power(token4, eight / 4, kD));
                const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (key4 + i < lo || key4 + i >= n) continue;      // what lies there may be anything
                    float x[8];
                    eight_floats(words[i], power_of(powers >> (8 * i) & 255u), x);
#pragma unroll
                    for (int h = 0; h < kRowsHeads; ++h) {
                        const float p = weight[wave][h][4 * run + i];
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[h][e] = fmaf(p, x[e], acc[h][e]);
                    }
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    // The lanes of an eight and the waves, in order.
    const bool poisoned = __any(unmapped);
#pragma unroll
    for (int h = 0; h < kRowsHeads; ++h) {
        if (poisoned) l[h] = __builtin_nanf("");
        if (l[h] != l[h]) m[h] = fmaxf(m[h], 0.f);              // (a result of NaN counts, whatever its maximum)
        if (lane == 0) part_m[wave][h] = m[h], part_l[wave][h] = l[h];
    }
    for (int s = 0; s < kSubs; ++s) {
        if (sub == s) {
#pragma unroll
            for (int h = 0; h < kRowsHeads; ++h)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float* to = &part[wave][h][eight * 8 + i];
                    *to = s == 0 ? acc[h][i] : *to + acc[h][i];
                }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < heads * kD; i += kRowsThreads) {
        const int h = i / kD, d = i % kD;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kRowsWaves; ++w) top = fmaxf(top, part_m[w][h]);
        float num = 0.f, den = 0.f;
#pragma unroll
        for (int w = 0; w < kRowsWaves; ++w) {
            const float by = part_m[w][h] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(part_m[w][h] - top);
            if (by > 0.f) num += part[w][h][d] * by;
            den += part_l[w][h] * by;
        }
        const long row_head = static_cast<long>(row) * q_heads + head0 + h;
        if (splits == 1) {
            out[row_head * kD + d] = from_float<T>(top == -INFINITY ? 0.f : num / den);
        } else {
            const long slot = row_head * splits + blockIdx.z;
            part_acc[slot * kD + d] = num;
            if (d == 0) part_ml[2 * slot] = top, part_ml[2 * slot + 1] = den;
        }
    }
}

// Merges the shares of a (row, query head) in their order: sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M).  A wave a row and head;
// lane s has share s's maximum and sum.
constexpr int kShares = kWave;
constexpr int kMergeThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kMergeThreads)
four_bit_merge_kernel(const float* __restrict__ part_acc, const float* __restrict__ part_ml, T* __restrict__ out, long row_heads, int dim, int splits) {
    const long row_head = static_cast<long>(blockIdx.x) * (kMergeThreads / kWave) + threadIdx.x / kWave;
    if (row_head >= row_heads) return;
    const int lane = threadIdx.x % kWave;
    const float m = lane < splits ? part_ml[2 * (row_head * splits + lane)] : -INFINITY;
    const float l = lane < splits ? part_ml[2 * (row_head * splits + lane) + 1] : 0.f;
    const float top = wave_max(m);
    const float by = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    const float den = wave_sum(m == -INFINITY ? 0.f : l * by);
    const bool mine = 4 * lane < dim;                            // (the other lanes go along: every lane's weight is asked for below)
    const int d = mine ? 4 * lane : 0;
    floatx4 num = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += 8) {
        floatx4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)                          // (a share behind the last is the last again and weighs nothing)
            x[i] = *reinterpret_cast<const floatx4*>(part_acc + (row_head * splits + min(s0 + i, splits - 1)) * dim + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float w = s0 + i < splits ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, by), s0 + i)) : 0.f;
            if (w > 0.f) {                                   // an empty share's sums were never written
#pragma unroll
                for (int e = 0; e < 4; ++e) num[e] += x[i][e] * w;
            }
        }
    }
    if (!mine) return;
    T* to = out + row_head * dim + d;
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = from_float<T>(top == -INFINITY ? 0.f : num[e] / den);
}

template <typename T>
static void merge_shares(const float* part_acc, const float* part_ml, void* out, int rows, int q_heads, int dim, int splits, hipStream_t stream) {
    const long row_heads = static_cast<long>(rows) * q_heads;
    four_bit_merge_kernel<T><<<ceil_div(row_heads, kMergeThreads / kWave), kMergeThreads, 0, stream>>>(part_acc, part_ml, static_cast<T*>(out), row_heads,
                                                                                                      dim, splits);
}

static FourBitPools read_pools(const void* k_codes, const void* k_powers, const void* v_codes, const void* v_powers, int pages) {
    auto bytes = [](const void* p) { return const_cast<uint8_t*>(static_cast<const uint8_t*>(p)); };
    return FourBitPools{bytes(k_codes), bytes(k_powers), bytes(v_codes), bytes(v_powers), pages};
}

}  // namespace leone

using namespace leone;

extern "C" int leone_four_bit_max_splits() { return kShares; }

extern "C" int leone_four_bit_attend_rows(const void* q, void* out, int dtype, const void* k_codes, const void* k_powers, const void* v_codes,
                                          const void* v_powers, int pages, const int* positions, const int* row_entry, const int* block_table,
                                          int max_blocks, int entries, int rows, int q_heads, int kv_heads, int head_dim, int page_tokens,
                                          float scale, int window, int splits, float* part_acc, float* part_ml, hipStream_t stream) {
    const char* what = "four_bit_attend_rows";
    const FourBitPools pools = read_pools(k_codes, k_powers, v_codes, v_powers, pages);
    if (check_four_bit(what, pools, kv_heads, head_dim, page_tokens, max_blocks)) return 1;
    LEONE_REQUIRE(q && out && positions && row_entry && block_table, "%s: null pointer", what);
    LEONE_REQUIRE(dtype == kF32 || dtype == kBF16, "%s: unknown type", what);
    LEONE_REQUIRE(rows > 0 && entries > 0 && q_heads > 0 && q_heads % kv_heads == 0, "%s: %d rows, %d entries, %d query heads over %d kv heads", what, rows,
                  entries, q_heads, kv_heads);
    LEONE_REQUIRE(window >= 0 && splits >= 1 && splits <= kShares, "%s: window %d must not be negative, splits %d in 1..%d", what, window, splits, kShares);
    LEONE_REQUIRE(splits == 1 || (part_acc && part_ml && reinterpret_cast<uintptr_t>(part_acc) % 16 == 0), "%s: %d shares need the workspace", what, splits);
    const int group = q_heads / kv_heads;
    const long tiles = static_cast<long>(kv_heads) * ((group + kRowsHeads - 1) / kRowsHeads);
    LEONE_REQUIRE(tiles <= 65535, "%s: too many heads for one launch", what);
    const dim3 grid(rows, static_cast<unsigned>(tiles), splits);
    const float to_log2 = scale * kLog2e;
#define LEONE_ROWS(N)                                                                                                                              \
    case N:                                                                                                                                        \
        if (dtype == kF32)                                                                                                                         \
            four_bit_attend_rows_kernel<N, float><<<grid, kRowsThreads, 0, stream>>>(                                                              \
                static_cast<const float*>(q), static_cast<float*>(out), pools, positions, row_entry, block_table, max_blocks, entries, q_heads,    \
                kv_heads, page_tokens, to_log2, window, splits, part_acc, part_ml);                                                                \
        else                                                                                                                                       \
            four_bit_attend_rows_kernel<N, bf16_t><<<grid, kRowsThreads, 0, stream>>>(                                                             \
                static_cast<const bf16_t*>(q), static_cast<bf16_t*>(out), pools, positions, row_entry, block_table, max_blocks, entries, q_heads,  \
                kv_heads, page_tokens, to_log2, window, splits, part_acc, part_ml);                                                                \
        break;
    switch (head_dim / kBlock) {
        LEONE_ROWS(1) LEONE_ROWS(2) LEONE_ROWS(3) LEONE_ROWS(4) LEONE_ROWS(5) LEONE_ROWS(6) LEONE_ROWS(7) LEONE_ROWS(8)
    }
#undef LEONE_ROWS
    LEONE_LAUNCH_CHECK(what);
    if (splits > 1) {
        if (dtype == kF32) merge_shares<float>(part_acc, part_ml, out, rows, q_heads, head_dim, splits, stream);
        else merge_shares<bf16_t>(part_acc, part_ml, out, rows, q_heads, head_dim, splits, stream);
        LEONE_LAUNCH_CHECK("four_bit_merge");
    }
    return 0;
}
