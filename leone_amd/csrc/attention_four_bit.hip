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
//    and, by a second product, the rest.  The eight bits of a bfloat16 are kept whole in elements down to 2^-14 of the row's largest;
//    smaller ones are off by up to 2^-22 of it.  Heads of 64 hold both parts in one product, the keys given twice.
//    The instruction adds eight neighbouring elements' products as multiples of 2^-13 of the power of two in the largest of them, cut
//    towards zero (measured; a product has six bits, so that what lies within 2^8 of the largest is whole), and the eights' sums in
//    float.  A score is off by less than 2^-10 of its eights' largest products, which seldom shows beside the weights' rounding: with every
//    eighth element of a query 512 times the others the mean error of a result is 9.6e-4, with float products 8.1e-4 (scores ten
//    wide, results of 0.63).
//  * the values are unpacked by the chip's own conversion, two to an instruction with their power, and brought from neighbouring
//    elements of a token to neighbouring tokens of an element by one byte permutation for two.  The second product is then
//    v_mfma_f32_16x16x32_bf16 on exact values; its weights are rounded to bfloat16, against a reference that is a whole number, so
//    that the rounding does not depend on how the keys are cut, and the sum is taken over the rounded weights.
// Operand layouts (lane l, c = l % 16, g = l / 16), checked on the chip: 4-bit operand: row c, elements 32 g .. + 31; 8-bit operand:
// column c, elements 16 g .. + 15 and 64 + 16 g .. + 15; a lane's power belongs to elements 32 g .. + 31 of its row or column.
// Result: column c, rows 4 g .. + 3.  A lane's scores of a tile's two halves are those of keys 4 g .. + 3 and 16 + 4 g .. + 3: it takes
// the values of the same keys (the second product may sum in any order), a run of four each, and the scores go into the second
// product as they are.  Every load of a wave is then of neighbouring bytes.
// The reference is raised only by a score that exceeds it by more than 8 (weights stay below 2^8): no exchange between lanes
// otherwise.
// Measured, heads of 128: 64 rows of 300 to 8,191 keys, 40 heads over 8, 64 us, 4.6 TB/s of a cache of 297 MB (a kernel
// that only reads it 47 to 55; 53 where the call before read the same); 8 rows of 8,176, 32 over 8, 17 us in 8 shares with their merge (71 MB; a plain read of it takes 13); one of
// 32,768, 64 over 8, 13.6 us in 32 (36 MB, 7); two of about 100 4.7 us, a trip to memory for every step from position to key.  Larger tiles, more
// tiles in flight and fewer waves a unit were level or slower (kTileKeys).
//
// ---- any shape and type ------------------------------------------------------------------------------------------------
// Float arithmetic of each key's elements by one lane: bound by instructions.  4 rows of 501 to 777 keys, 16 heads over 4, float32:
// 14.2 us with the merge.
#include "common.h"
#include "four_bit_attend.h"
#include "leone_hip.h"
#include "score_shape.h"

#include <math.h>
#include <type_traits>

namespace leone {

// Query heads a workgroup of the decode kernel takes: a product has sixteen columns; wide heads' sums take the room of eight.
__host__ __device__ constexpr int decode_columns(int dim) { return dim <= 128 ? 16 : 8; }

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
    const int all = entry >= 0 && entry < entries ? min(positions[row], kLastPosition) + 1 : 0;
    const int lo = first_key(max(all - 1, 0), window, 0);
    const int n = min(all, max_blocks * page_tokens);            // keys behind the block table's reach have no page
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
    bool unmapped = n < all;
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
            num += part[w][h][d] * by;                          // (a NaN value stays one however little it weighs)
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

// ---- single tokens on the matrix cores -----------------------------------------------------------------------------------
constexpr int kDecodeWaves = 4;
constexpr int kDecodeThreads = kDecodeWaves * kWave;
constexpr int kTileKeys = 32;     // (of 64 a lone wave is a fifth faster, but two a SIMD fit instead of three: 64 rows of 300 to 8,191 keys level, 2 of 100 10 % slower)

template <int kD, bool kOnePage>
__global__ void __launch_bounds__(kDecodeThreads, kD <= 128 ? 3 : 2)
four_bit_decode_kernel(const bf16_t* __restrict__ q, bf16_t* __restrict__ out, FourBitPools pools, const int* __restrict__ positions,
                       const int* __restrict__ row_entry, const int* __restrict__ block_table, int max_blocks, int entries, int q_heads,
                       int kv_heads, int page_shift, float to_log2, int window, int splits, float* __restrict__ part_acc,
                       float* __restrict__ part_ml) {
    constexpr int kCols = decode_columns(kD);
    constexpr int kSubs = kTileKeys / 16;                         // products of sixteen keys a tile
    constexpr int kSteps = kD <= 128 ? 1 : kD / 128;              // of 128 elements
    constexpr int kParts = kD <= 64 ? 1 : 2;                      // products a step: heads of 64 hold both parts of a query in one
    constexpr int kVLoads = kD <= 128 ? 1 : kD / 128;             // eights a lane has of each of its tokens
    constexpr int kDepth = 2;
    constexpr int kOwn = kD / 16;                                 // elements a lane has of each of its tokens
    extern __shared__ float smem[];                               // [waves][columns][kD], then maxima and sums

    const int group = q_heads / kv_heads, col_tiles = (group + kCols - 1) / kCols;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int c = lane & 15, g = lane >> 4;
    // Rows differ in length, and a unit whose two workgroups are long ones is what the launch waits for: workgroups 256 apart share a unit, and
    // with the rows of every second half of the heads in falling order they are two rows', not two heads' of one (64 rows of 300
    // to 8,191 keys in no order, 8 kv heads: 63.8 us, 70.7 in the grid's order).
    const int row = blockIdx.y >= gridDim.y / 2 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const int kvh = blockIdx.y / col_tiles, col0 = (blockIdx.y - kvh * col_tiles) * kCols;
    const int cols = min(kCols, group - col0), split = blockIdx.z;
    const int entry = row_entry[row], pos = positions[row];
    const int all = entry >= 0 && entry < entries ? min(pos, kLastPosition) + 1 : 0;
    const int lo = first_key(max(all - 1, 0), window, 0);
    const int n = min(all, max_blocks << page_shift);             // keys behind the block table's reach have no page
    const int* table = block_table + static_cast<long>(entry) * max_blocks;
    const int t_begin = lo / kTileKeys, t_end = (n + kTileKeys - 1) / kTileKeys;
    const int share = (t_end - t_begin + splits - 1) / splits;
    const int my_begin = t_begin + split * share, my_end = min(my_begin + share, t_end);
    const int page_tokens = 1 << page_shift, page_mask = page_tokens - 1;
    const long code_bytes = four_bit_codes(page_tokens, kD), power_bytes = four_bit_powers(page_tokens, kD);

    // A tile: the page ids of its halves of sixteen keys (of the whole tile, where pages hold 32 or more: kOnePage) come by scalar loads,
    // which are waited for apart from the others, then its bytes.  What has no page is read from the first one and masked later.
    // (Every call of `issue` is the same loads whatever the tile, also behind the last: after a load that may or may not have been
    // issued the compiler waits for all.  Addresses are a base that is the same for the wave and a lane's 32-bit offset that does not
    // change: with 64-bit products for every load a tile cost 1,700 cycles of a wave, half of it scalar arithmetic.)
    constexpr int kPages = kOnePage ? 1 : kSubs;
    struct Tile {
        uint4 k[kSubs][kSteps];                                   // key 16 sub + c
        unsigned k_power[kSubs][kSteps];
        uint4 v[kSubs][kVLoads];                                  // keys 16 sub + 4 g .. + 3
        unsigned v_power[kSubs][kVLoads];
        int page[kPages];
    };
    struct Pages {
        int id[kPages];
    };
    const int k_block = kD <= 64 ? g & 1 : g, eight = kD <= 64 ? c >> 1 : c;           // the lane's first block and eight
    const unsigned k_code_at = four_bit_key(c, k_block, page_tokens), k_power_at = four_bit_key_power(c, k_block, kD);
    const unsigned v_code_at = four_bit_value(4 * g, eight, kD), v_power_at = four_bit_value_power(4 * g, eight / 4, kD);
    const unsigned code_stride = static_cast<unsigned>(code_bytes) * kv_heads, power_stride = static_cast<unsigned>(power_bytes) * kv_heads;
    const uint8_t* k_codes = pools.k_codes + kvh * code_bytes;
    const uint8_t* k_powers = pools.k_powers + kvh * power_bytes;
    const uint8_t* v_codes = pools.v_codes + kvh * code_bytes;
    const uint8_t* v_powers = pools.v_powers + kvh * power_bytes;
    auto find = [&](int t) {
        Pages found;
#pragma unroll
        for (int i = 0; i < kPages; ++i) found.id[i] = table[min((t * kTileKeys + 16 * i) >> page_shift, max_blocks - 1)];
        return found;
    };
    auto issue = [&](int t, const Pages& found, Tile& r) {
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub) {
            const int i = kOnePage ? 0 : sub;
            r.page[i] = found.id[i];
            const unsigned page = static_cast<unsigned>(found.id[i]) < static_cast<unsigned>(pools.pages) ? found.id[i] : 0;
            const unsigned token = (t * kTileKeys + 16 * sub) & page_mask;
            const unsigned long long codes = static_cast<unsigned long long>(page) * code_stride, powers = static_cast<unsigned long long>(page) * power_stride;
            const uint8_t* kc = k_codes + codes + 16 * token;                             // (a block of so many tokens' keys)
            const uint8_t* kp = k_powers + powers + kD / kBlock * token;
            const uint8_t* vc = v_codes + codes + kD / 2 * token;
            const uint8_t* vp = v_powers + powers + kD / kBlock * token;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                r.k[sub][s] = load_streamed16(kc + (k_code_at + s * four_bit_key(0, 4, page_tokens)));
                r.k_power[sub][s] = kp[k_power_at + 4 * s];
            }
#pragma unroll
            for (int s = 0; s < kVLoads; ++s) {
                r.v[sub][s] = load_streamed16(vc + (v_code_at + s * four_bit_value(0, 16, kD)));
                r.v_power[sub][s] = *reinterpret_cast<const unsigned*>(vp + (v_power_at + s * four_bit_value_power(0, 4, kD)));
            }
        }
    };

    int t = my_begin + wave;
    Pages ahead{};
    if (t < my_end) ahead = find(t);

    // The query, column c: elements 16 g .. + 15 and 64 + 16 g .. + 15 of every 128, in two parts.
    intx8 query[kSteps][kParts];
    int power_high, power_low;
    {
        const bf16_t* from = q + (static_cast<long>(row) * q_heads + kvh * group + col0 + (c < cols ? c : 0)) * kD + 16 * g;
        constexpr int kRuns = kD <= 64 ? 1 : 2;
        uint4 raw[kSteps][kRuns][2];
        unsigned top = 0;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int run = 0; run < kRuns; ++run)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    raw[s][run][i] = c < cols ? *reinterpret_cast<const uint4*>(from + 128 * s + 64 * run + 8 * i) : uint4{0u, 0u, 0u, 0u};
                    top = largest_bits(raw[s][run][i], top);
                }
        auto larger = [](unsigned a, unsigned b) { return max(a, b); };
        top = join_lanes<16>(top, larger);
        top = join_lanes<32>(top, larger);
        const int power = query_power(top);
        const float unit = query_unit(power);
        power_high = power, power_low = rest_power(power);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            int high[2][4], low[2][4];
#pragma unroll
            for (int run = 0; run < kRuns; ++run) two_parts(raw[s][run], unit, high[run], low[run]);
            if constexpr (kD <= 64) {
                query[s][0] = intx8{high[0][0], high[0][1], high[0][2], high[0][3], low[0][0], low[0][1], low[0][2], low[0][3]};
            } else {
                query[s][0] = intx8{high[0][0], high[0][1], high[0][2], high[0][3], high[1][0], high[1][1], high[1][2], high[1][3]};
                query[s][1] = intx8{low[0][0], low[0][1], low[0][2], low[0][3], low[1][0], low[1][1], low[1][2], low[1][3]};
            }
        }
        if constexpr (kD <= 64) {
            if (g >= 2) power_high = power_low;                   // the second two blocks are the keys against the rest
        }
    }

    float m_ref = -INFINITY, l_run = 0.f;
    bool unmapped = n < all;
    floatx4 acc[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};

    auto finish = [&](int tile, Tile& r) {
        const int key0 = tile * kTileKeys;
        bool no_page[kSubs], full = key0 >= lo && key0 + kTileKeys <= n;          // the same for the whole wave
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub) {
            no_page[sub] = static_cast<unsigned>(r.page[kOnePage ? 0 : sub]) >= static_cast<unsigned>(pools.pages);
            full &= !no_page[sub];
        }
        // ---- scores of keys 16 sub + 4 g .. + 3 for column c
        floatx4 s4[kSubs];
#pragma unroll
        for (int sub = 0; sub < kSubs; ++sub) s4[sub] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int part = 0; part < kParts; ++part)             // (the sixteens in turn: no product waits for the one before)
#pragma unroll
                for (int sub = 0; sub < kSubs; ++sub)
                    s4[sub] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(low_half(r.k[sub][s]), query[s][part], s4[sub], 4, 0, 0,
                                                                              static_cast<int>(r.k_power[sub][s]), 0, part == 0 ? power_high : power_low);
        float sc[4 * kSubs];
#pragma unroll
        for (int j = 0; j < 4 * kSubs; ++j) sc[j] = s4[j / 4][j % 4];
        if (!full) {
#pragma unroll
            for (int sub = 0; sub < kSubs; ++sub) {
                unmapped |= no_page[sub] && key0 + 16 * sub < n && key0 + 16 * sub + 16 > lo;
                unsigned hidden = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = key0 + 16 * sub + 4 * g + i;
                    if (no_page[sub] || key < lo || key >= n) sc[4 * sub + i] = -INFINITY, hidden |= 0xffu << (8 * i);
                }
                // what lies in places out of sight may be anything: a power of one makes it a number
#pragma unroll
                for (int s = 0; s < kVLoads; ++s) r.v_power[sub][s] = (r.v_power[sub][s] & ~hidden) | (0x7f7f7f7fu & hidden);
            }
        }
        float top = sc[0];
#pragma unroll
        for (int j = 1; j < 4 * kSubs; ++j) top = fmaxf(top, sc[j]);
        top *= to_log2;
        if (__any(top > m_ref + kRaise)) {                        // -inf + 8 is -inf: the first scores always raise
            top = max_lanes<16>(top);
            top = max_lanes<32>(top);
            const float m_new = fmaxf(m_ref, ceilf(top));
            const float keep = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_ref - m_new);
            m_ref = m_new;
            l_run *= keep;
#pragma unroll
            for (int j = 0; j < kOwn; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[j][v] *= keep;
        }
        const float shift = m_ref == -INFINITY ? 0.f : -m_ref;
#pragma unroll
        for (int two = 0; two < kSubs / 2; ++two) {               // 32 keys of the second product
            bf16x8 pt;
#pragma unroll
            for (int j = 0; j < 8; ++j) pt[j] = static_cast<__bf16>(__builtin_amdgcn_exp2f(fmaf(sc[8 * two + j], to_log2, shift)));
            {
                const uint4 packed = __builtin_bit_cast(uint4, pt);
                const unsigned pairs[4] = {packed.x, packed.y, packed.z, packed.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    l_run = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pairs[i]), __builtin_bit_cast(bf16x2, 0x3f803f80u), l_run, false);
            }
            // ---- values: the lane's elements of its eight tokens, two elements at a time from every token, then by element
#pragma unroll
            for (int s = 0; s < kVLoads; ++s) {
                unsigned words[8];
                float power[8];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 raw = r.v[2 * two + half][s];
                    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        words[4 * half + i] = kD <= 64 ? w[i] >> (16 * (c & 1)) : w[i];
                        power[4 * half + i] = power_of(r.v_power[2 * two + half][s] >> (8 * i) & 255u);
                    }
                }
                auto pair = [&](auto index) {
                    constexpr int i = decltype(index)::value;
                    unsigned both[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) both[k] = two_bf16<i>(words[k], power[k]);
                    uint4 even, odd;
                    even.x = __builtin_amdgcn_perm(both[1], both[0], 0x05040100u), odd.x = __builtin_amdgcn_perm(both[1], both[0], 0x07060302u);
                    even.y = __builtin_amdgcn_perm(both[3], both[2], 0x05040100u), odd.y = __builtin_amdgcn_perm(both[3], both[2], 0x07060302u);
                    even.z = __builtin_amdgcn_perm(both[5], both[4], 0x05040100u), odd.z = __builtin_amdgcn_perm(both[5], both[4], 0x07060302u);
                    even.w = __builtin_amdgcn_perm(both[7], both[6], 0x05040100u), odd.w = __builtin_amdgcn_perm(both[7], both[6], 0x07060302u);
                    acc[8 * s + 2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, even), pt, acc[8 * s + 2 * i], 0, 0, 0);
                    acc[8 * s + 2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, odd), pt, acc[8 * s + 2 * i + 1], 0, 0, 0);
                };
                pair(std::integral_constant<int, 0>{});
                pair(std::integral_constant<int, 1>{});
                if constexpr (kD > 64) {
                    pair(std::integral_constant<int, 2>{});
                    pair(std::integral_constant<int, 3>{});
                }
            }
        }
    };

    // kDepth tiles in turn: a wave always has loads in flight.
    Tile ring[kDepth];
    if (t < my_end) {
#pragma unroll
        for (int i = 0; i < kDepth - 1; ++i) {
            issue(t + i * kDecodeWaves, ahead, ring[i]);
            ahead = find(t + (i + 1) * kDecodeWaves);
        }
        bool more = true;
        while (more) {
#pragma unroll
            for (int i = 0; i < kDepth; ++i) {
                issue(t + (kDepth - 1) * kDecodeWaves, ahead, ring[(i + kDepth - 1) % kDepth]);
                ahead = find(t + kDepth * kDecodeWaves);
                finish(t, ring[i]);
                t += kDecodeWaves;
                if (t >= my_end) {
                    more = false;
                    break;
                }
            }
        }
    }

    // ---- the four waves, in their order
    float* sm_acc = smem;
    float* sm_m = smem + kDecodeWaves * cols * kD;
    float* sm_l = sm_m + kDecodeWaves * cols;
    l_run = add_lanes<16>(l_run);
    l_run = add_lanes<32>(l_run);
    if (unmapped) l_run = __builtin_nanf("");
    if (l_run != l_run) m_ref = fmaxf(m_ref, 0.f);                // (a result of NaN counts, whatever its maximum)
    if (c < cols) {
        if (g == 0) sm_m[wave * cols + c] = m_ref, sm_l[wave * cols + c] = l_run;
        // register v of sum j is, in row 4 g + v, element j of that lane's own
        float* to = sm_acc + (wave * cols + c) * kD;
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int j = 0; j < kOwn; j += 4) {
                const int d = kD <= 64 ? 4 * (4 * g + v) + j : 128 * (j / 8) + 8 * (4 * g + v) + j % 8;
                *reinterpret_cast<floatx4*>(to + d) = floatx4{acc[j][v], acc[j + 1][v], acc[j + 2][v], acc[j + 3][v]};
            }
    }
    __syncthreads();
    for (int i = threadIdx.x * 4; i < cols * kD; i += kDecodeThreads * 4) {
        const int col = i / kD, d = i % kD;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kDecodeWaves; ++w) top = fmaxf(top, sm_m[w * cols + col]);
        floatx4 num = {0.f, 0.f, 0.f, 0.f};
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < kDecodeWaves; ++w) {
            const float mw = sm_m[w * cols + col];
            const float by = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - top);
            const floatx4 part = *reinterpret_cast<const floatx4*>(&sm_acc[(w * cols + col) * kD + d]);
#pragma unroll
            for (int e = 0; e < 4; ++e) num[e] += part[e] * by;
            den += sm_l[w * cols + col] * by;
        }
        const long row_head = static_cast<long>(row) * q_heads + kvh * group + col0 + col;
        if (splits == 1) {
            const float inv = top == -INFINITY ? 0.f : 1.f / den;   // a row that sees nothing: zeros
            uint2 packed;
            packed.x = bf16_bits_from_float(num[0] * inv) | static_cast<unsigned>(bf16_bits_from_float(num[1] * inv)) << 16;
            packed.y = bf16_bits_from_float(num[2] * inv) | static_cast<unsigned>(bf16_bits_from_float(num[3] * inv)) << 16;
            *reinterpret_cast<uint2*>(out + row_head * kD + d) = packed;
        } else {
            const long slot = row_head * splits + split;
            *reinterpret_cast<floatx4*>(part_acc + slot * kD + d) = num;
            if (d == 0) part_ml[2 * slot] = top, part_ml[2 * slot + 1] = den;
        }
    }
}

// The merge of shares.  kGroup neighbouring lanes have a row and head, four elements each; between them they hold the shares' maxima and
// sums and hand the weights round, four shares' sums on their way at a time.  (A merge of its own beside those of attention_merge.h: they
// give bfloat16 alone; the one over rows multiplies the sums of every share, also of those that the prompt kernel never wrote, and the
// one over tiles leaves out what weighs nothing, a NaN with it.)
constexpr int kMergeThreads = 256;
constexpr int kMergeAhead = 4;
constexpr float kNotWritten = -1.f;                              // in a weight's place: a share of no keys, whose sums may be anything

template <int kGroup, typename T>
__global__ void __launch_bounds__(kMergeThreads)
four_bit_merge_kernel(const float* __restrict__ part_acc, const float* __restrict__ part_ml, T* __restrict__ out, long items, int q_heads, int dim,
                      int splits, const int* __restrict__ tiles, int limit) {
    constexpr int kEach = kShares / kGroup;                      // shares whose weights a lane holds
    const int lane = threadIdx.x % kGroup;
    long item = (static_cast<long>(blockIdx.x) * kMergeThreads + threadIdx.x) / kGroup;
    bool exists = item < items;
    if (!exists) item = 0;                                       // (every lane goes along: weights are handed round)
    if (tiles != nullptr) {
        const long place = item / q_heads;
        const int* tile = tiles + 3 * (place / kTileRows);
        const int r = static_cast<int>(place % kTileRows);
        exists &= r < tile[2] && tile[1] >= 0 && tile[1] < limit - r;
        item = exists ? (static_cast<long>(tile[1]) + r) * q_heads + item % q_heads : 0;
    }
    const float* ml = part_ml + 2 * item * splits;
    float m[kEach], by[kEach], top = -INFINITY, den = 0.f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        m[k] = k * kGroup + lane < splits ? ml[2 * (k * kGroup + lane)] : -INFINITY;
        by[k] = k * kGroup + lane < splits ? ml[2 * (k * kGroup + lane) + 1] : 0.f;
        top = fmaxf(top, m[k]);
    }
    top = join_span<kGroup>(top, [](float a, float b) { return fmaxf(a, b); });
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const float w = m[k] == -INFINITY ? kNotWritten : __builtin_amdgcn_exp2f(m[k] - top);
        den += m[k] == -INFINITY ? 0.f : by[k] * w;
        by[k] = w;
    }
    den = join_span<kGroup>(den, [](float a, float b) { return a + b; });
    const bool mine = 4 * lane < dim;
    const float* from = part_acc + item * splits * dim + (mine ? 4 * lane : 0);
    floatx4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        for (int s0 = k * kGroup; s0 < min(splits, (k + 1) * kGroup); s0 += kMergeAhead) {
            floatx4 x[kMergeAhead];
#pragma unroll
            for (int i = 0; i < kMergeAhead; ++i)                // (a share behind the last is the last again and weighs nothing)
                x[i] = *reinterpret_cast<const floatx4*>(from + static_cast<long>(min(s0 + i, splits - 1)) * dim);
#pragma unroll
            for (int i = 0; i < kMergeAhead; ++i) {              // (a weight that underflows is no reason: a NaN value stays one)
                const float w = s0 + i < splits ? __shfl(by[k], (s0 + i) % kGroup, kGroup) : kNotWritten;
#pragma unroll
                for (int e = 0; e < 4; ++e) num[e] = w == kNotWritten ? num[e] : fmaf(x[i][e], w, num[e]);
            }
        }
    }
    if (!exists || !mine) return;
    T* to = out + item * dim + 4 * lane;
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = from_float<T>(top == -INFINITY ? 0.f : num[e] / den);
}

template <typename T>
static void launch_merge(const float* part_acc, const float* part_ml, T* out, long items, int q_heads, int dim, int splits, const int* tiles,
                         int limit, hipStream_t stream) {
#define LEONE_MERGE(GROUP)                                                                                                                    \
    four_bit_merge_kernel<GROUP, T><<<ceil_div(items * GROUP, kMergeThreads), kMergeThreads, 0, stream>>>(part_acc, part_ml, out, items, q_heads, \
                                                                                                         dim, splits, tiles, limit)
    if (dim <= 64) LEONE_MERGE(16);
    else if (dim <= 128) LEONE_MERGE(32);
    else LEONE_MERGE(64);
#undef LEONE_MERGE
}

void merge_four_bit_shares(const float* part_acc, const float* part_ml, void* out, int dtype, long rows, int q_heads, int dim, int splits,
                           const int* tiles, int limit, hipStream_t stream) {
    const long items = rows * q_heads;
    if (dtype == kF32) launch_merge(part_acc, part_ml, static_cast<float*>(out), items, q_heads, dim, splits, tiles, limit, stream);
    else launch_merge(part_acc, part_ml, static_cast<bf16_t*>(out), items, q_heads, dim, splits, tiles, limit, stream);
}

}  // namespace leone

using namespace leone;

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
    LEONE_REQUIRE(scale > 0.f, "%s: the score scale must be positive", what);
    LEONE_REQUIRE(window >= 0 && splits >= 1 && splits <= kShares, "%s: window %d must not be negative, splits %d in 1..%d", what, window, splits, kShares);
    LEONE_REQUIRE(splits == 1 || (part_acc && part_ml && reinterpret_cast<uintptr_t>(part_acc) % 16 == 0), "%s: %d shares need the workspace", what, splits);
    LEONE_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0, "%s: queries and results start at multiples of 16 bytes", what);
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
        merge_four_bit_shares(part_acc, part_ml, out, dtype, rows, q_heads, head_dim, splits, nullptr, rows, stream);
        LEONE_LAUNCH_CHECK("four_bit_merge");
    }
    return 0;
}

extern "C" int leone_four_bit_decode(const void* q, void* out, const void* k_codes, const void* k_powers, const void* v_codes, const void* v_powers,
                                     int pages, const int* positions, const int* row_entry, const int* block_table, int max_blocks, int entries,
                                     int rows, int q_heads, int kv_heads, int head_dim, int page_tokens, float scale, int window, int splits,
                                     float* part_acc, float* part_ml, hipStream_t stream) {
    const char* what = "four_bit_decode";
    const FourBitPools pools = read_pools(k_codes, k_powers, v_codes, v_powers, pages);
    if (check_four_bit(what, pools, kv_heads, head_dim, page_tokens, max_blocks)) return 1;
    LEONE_REQUIRE(q && out && positions && row_entry && block_table, "%s: null pointer", what);
    LEONE_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "%s: heads of 64, 128 or 256 elements, not %d", what, head_dim);
    LEONE_REQUIRE(page_tokens >= 16 && (page_tokens & (page_tokens - 1)) == 0, "%s: pages of a power of two tokens from 16 on, not %d", what, page_tokens);
    LEONE_REQUIRE(rows > 0 && entries > 0 && q_heads > 0 && q_heads % kv_heads == 0, "%s: %d rows, %d entries, %d query heads over %d kv heads", what, rows,
                  entries, q_heads, kv_heads);
    LEONE_REQUIRE(scale > 0.f, "%s: the score scale must be positive", what);
    LEONE_REQUIRE(window >= 0 && splits >= 1 && splits <= kShares, "%s: window %d must not be negative, splits %d in 1..%d", what, window, splits, kShares);
    LEONE_REQUIRE(splits == 1 || (part_acc && part_ml && reinterpret_cast<uintptr_t>(part_acc) % 16 == 0), "%s: %d shares need the workspace", what, splits);
    LEONE_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0, "%s: queries and results start at multiples of 16 bytes", what);
    const int group = q_heads / kv_heads, columns = decode_columns(head_dim);
    const long tiles = static_cast<long>(kv_heads) * ((group + columns - 1) / columns);
    LEONE_REQUIRE(tiles <= 65535, "%s: too many heads for one launch", what);
    LEONE_REQUIRE(four_bit_codes(page_tokens, head_dim) * kv_heads < 0x7fffffffL, "%s: a page of %d heads is too large", what, kv_heads);
    const dim3 grid(rows, static_cast<unsigned>(tiles), splits);
    const int cols = group < columns ? group : columns;
    const size_t shared = static_cast<size_t>(kDecodeWaves) * cols * (head_dim + 2) * sizeof(float);
    int page_shift = 0;
    while ((1 << page_shift) < page_tokens) ++page_shift;
    const float to_log2 = scale * kLog2e;
#define LEONE_DECODE_CALL(D, ONE)                                                                                                          \
    four_bit_decode_kernel<D, ONE><<<grid, kDecodeThreads, shared, stream>>>(                                                              \
        static_cast<const bf16_t*>(q), static_cast<bf16_t*>(out), pools, positions, row_entry, block_table, max_blocks, entries, q_heads,  \
        kv_heads, page_shift, to_log2, window, splits, part_acc, part_ml)
#define LEONE_DECODE(D)                                           \
    do {                                                          \
        if (page_tokens >= kTileKeys) LEONE_DECODE_CALL(D, true); \
        else LEONE_DECODE_CALL(D, false);                         \
    } while (0)
    if (head_dim == 64) LEONE_DECODE(64);
    else if (head_dim == 128) LEONE_DECODE(128);
    else LEONE_DECODE(256);
#undef LEONE_DECODE
#undef LEONE_DECODE_CALL
    LEONE_LAUNCH_CHECK(what);
    if (splits > 1) {
        merge_four_bit_shares(part_acc, part_ml, out, kBF16, rows, q_heads, head_dim, splits, nullptr, rows, stream);
        LEONE_LAUNCH_CHECK("four_bit_merge");
    }
    return 0;
}
