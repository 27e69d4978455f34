// Causal attention of prompt portions over the cache of 4 bits an element (four_bit.h) on the matrix cores, bfloat16, heads of 64 and
// 128.
//
// A wave takes a tile of 32 consecutive rows of one request and one query head, a workgroup four tiles of the request (the host lists
// them: entry, first row, rows); it walks the keys its tiles can see once, 64 at a time.  Keys go from the cache to shared memory and
// into the first product as they are:
// v_mfma_scale_f32_32x32x64_f8f6f4, 4-bit keys with their powers against queries in two 8-bit parts (see attention_four_bit.hip).  It takes as
// long as the bfloat16 product of the same size would, but a wave reads a quarter of the bytes from shared memory, which four waves
// with 32 rows each read all keys from.  Values are unpacked once for the four waves: a thread has four tokens of eight elements
// in flight while a stage is worked on, turns them into runs of eight tokens of one element and leaves them in shared memory for
// the next, in bfloat16, where v_mfma_f32_32x32x16_bf16 takes them.  Both come by way of registers, asked for two stages ahead: loads
// that write to shared memory themselves are waited for before it is read again.
//
// 2,048 rows behind 8,192 tokens, 32 heads of 128 over 8: 276 to 284 us among other calls, 304 to 312 over and over on the same inputs; at 281
// 1,100 TFLOP/s of the exact work (a product of two 8,192-square bfloat16 matrices reaches 1,200 by the vendor library, the bfloat16 prompt
// kernel 933 here); 128 rows behind 30,720, 64 heads: 131 to 143 us in 8 ranges and their merge, 8 of them.  A pass of 32 keys is 512 cycles of the matrix cores and 560 of vector instructions (a weight is an
// exponential, a value a conversion and a permutation), and the two waves of a SIMD overlap them in part: the matrix cores are busy 45 %
// of the time, the vector units 47 %.  Forcing the overlap does not pay: two heads a workgroup, four waves a phase behind the other four
// with a barrier a phase 382 us; a pass's products asked for before the last one's weights 321; two heads a wave 481.
//
// Operand layouts (lane l, j = l % 32, h = l / 32): 4-bit operand: row j, elements 32 h .. + 31; 8-bit operand: column j, elements 16 h ..
// + 15 and 32 + 16 h .. + 15; a lane's power belongs to elements 32 h .. + 31 of its row or column; result: column j, rows
// 8 (v / 4) + 4 h + v % 4 in register v.  Row r of a pass's 32 keys is key r with bits 2 and 3 swapped: a lane's scores are
// those of keys 8 h .. + 7 and 16 + 8 h .. + 7 and go into the second product as they are.  Element d of the values is
// in place (d % 8) (dim / 8) + d / 8 of a run's row, so that neighbouring lanes, which have neighbouring eights, write neighbouring
// places; a lane's results are then eight neighbouring elements at a time.
//
// Softmax in powers of two against a reference that is a whole number and is raised only by a score that exceeds it by more than 8; the
// sum is taken over the rounded weights.  Few rows over many keys: the keys are cut into `splits` ranges of whole stages, a
// workgroup each, merged by a second kernel.
// A NaN value counts for the rows that see it only: a tile's rows see different keys, and a weight of zero would not keep it out, so
// that such a block is left as zeros in shared memory, its key is noted, and the rows in whose sight it is are made NaN.
#include "common.h"
#include "four_bit_attend.h"
#include "leone_hip.h"
#include "prefill_order.h"
#include "score_shape.h"

#include <math.h>
#include <type_traits>

namespace leone {

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float floatx16;

constexpr int kPromptWaves = 4;
constexpr int kPromptThreads = kPromptWaves * kWave;
constexpr int kStageKeys = 64;
constexpr int kPassKeys = 32;
constexpr int kMaxRanges = 32;

// Row of a pass's first product <-> key of the pass.
__device__ inline int pass_key(int x) { return (x & 0x13) | ((x & 4) << 1) | ((x & 8) >> 1); }

// A barrier that orders shared memory alone: __syncthreads waits for every load in flight, the stages that are on their way among them.
__device__ inline void shared_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int kD>
struct PromptStage {
    uint4 keys[kD / kBlock * kStageKeys];             // [half][block][row of the first product]
    uint4 values[8 * kD];                             // [run of eight tokens][place of the element]
};

// kWide: a stage's keys lie on one page, whose id is the same for the workgroup.
template <int kD, bool kWide>
__global__ void __launch_bounds__(kPromptThreads, 2)
four_bit_prefill_kernel(const bf16_t* __restrict__ q, bf16_t* __restrict__ out, FourBitPools pools, const int* __restrict__ positions,
                        const int* __restrict__ tiles, int n_groups, int rows, const int* __restrict__ block_table, int max_blocks, int entries,
                        int q_heads, int kv_heads, int page_shift, float to_log2, int window, int splits, float* __restrict__ part_acc,
                        float* __restrict__ part_ml) {
    constexpr int kBlocks = kD / kBlock;              // blocks of a vector
    constexpr int kSteps = kD / 64;                   // of the first product
    constexpr int kDT = kD / 32;                      // 32-row tiles of the second product's result
    constexpr int kEights = kD / 8;
    constexpr int kKeyUnits = kBlocks * kStageKeys;   // sixteen-byte units of a stage's keys, and of its values
    static_assert(kKeyUnits <= kPromptThreads, "a thread brings at most one unit of keys and one of values");
    __shared__ PromptStage<kD> stages[2];
    // Keys whose value block is NaN, of three stages in turn: one is read, one written and one cleared between two barriers.
    __shared__ unsigned long long nan_keys[3][kBlocks];
    __shared__ int nan_seen[3];
    __shared__ int wave_lo[kPromptWaves], wave_hi[kPromptWaves];
    __shared__ int unmapped_seen;

    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
    const int j = lane & 31, h = lane >> 5;
    const PrefillWork work = prefill_work(static_cast<int>(blockIdx.x), q_heads, n_groups);
    const int head = work.head, kvh = head / (q_heads / kv_heads);
    const int page_tokens = 1 << page_shift, page_mask = page_tokens - 1;
    const int* my_tile = tiles + 3 * (static_cast<long>(work.group) * kPromptWaves + wave);
    const int entry = tiles[3 * static_cast<long>(work.group) * kPromptWaves];
    // (rows that are not there, or that the workspace has no room for, are no tile's)
    const int tile_row0 = my_tile[1], wave_rows = tile_row0 < 0 ? 0 : min(min(my_tile[2], kTileRows), rows - tile_row0);
    const bool entry_ok = entry >= 0 && entry < entries;
    const int p0 = wave_rows > 0 ? min(positions[tile_row0], kLastPosition) : 0;     // a tile's rows stand at consecutive positions
    const int p_last = p0 + wave_rows - 1;
    const int reach = max_blocks << page_shift;                  // keys behind it have no page
    const int key_hi = wave_rows > 0 && entry_ok ? min(p_last + 1, reach) : 0;      // keys the wave may read: [key_lo, key_hi)
    const int key_lo = first_key(max(p0, 0), window, 0);
    const int full_hi = p0 + 1, full_lo = wave_rows > 0 ? first_key(p_last, window, 0) : 0;    // keys that every row of the wave sees
    if (lane == 0) {
        wave_lo[wave] = key_hi > key_lo ? key_lo : 0x7fffffff;
        wave_hi[wave] = key_hi > key_lo ? key_hi : 0;
    }
    if (tid == 0) unmapped_seen = 0;
    if (tid < 3 * kBlocks) nan_keys[tid / kBlocks][tid % kBlocks] = 0;
    if (tid < 3) nan_seen[tid] = 0;
    __syncthreads();
    if (wave_rows > 0 && entry_ok && p_last >= reach) unmapped_seen = 1;
    int group_lo = 0x7fffffff, group_hi = 0;
#pragma unroll
    for (int w = 0; w < kPromptWaves; ++w) group_lo = min(group_lo, wave_lo[w]), group_hi = max(group_hi, wave_hi[w]);
    if (splits > 1 && group_hi > group_lo) {
        const int s_begin = group_lo / kStageKeys, s_end = (group_hi + kStageKeys - 1) / kStageKeys;
        const int share = (s_end - s_begin + splits - 1) / splits;
        const int mine_lo = (s_begin + static_cast<int>(blockIdx.y) * share) * kStageKeys;
        group_lo = max(group_lo, mine_lo);
        group_hi = min(group_hi, mine_lo + share * kStageKeys);
    }
    const bool row_ok = j < wave_rows;
    const int row_pos = row_ok && entry_ok ? p0 + j : -1;        // -1: the row sees no key
    const int row_lo = first_key(max(row_pos, 0), window, 0);

    float m_ref = -INFINITY, l_run = 0.f;
    floatx16 acc[kDT];
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[dt][v] = 0.f;

    if (group_hi > group_lo) {                                   // (the same for the workgroup)
        // The query, column j: elements 16 h .. + 15 and 32 + 16 h .. + 15 of every 64, in two parts.
        intx8 query[kSteps][2];
        int power_high, power_low;
        {
            const bf16_t* from = q + (static_cast<long>(tile_row0 + (row_ok ? j : 0)) * q_heads + head) * kD + 16 * h;
            uint4 raw[kSteps][2][2];
            unsigned top = 0;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int run = 0; run < 2; ++run)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        raw[s][run][i] = row_ok ? *reinterpret_cast<const uint4*>(from + 64 * s + 32 * run + 8 * i) : uint4{0u, 0u, 0u, 0u};
                        top = largest_bits(raw[s][run][i], top);
                    }
            top = join_lanes<32>(top, [](unsigned a, unsigned b) { return max(a, b); });
            power_high = query_power(top), power_low = rest_power(power_high);
            const float unit = query_unit(power_high);
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                int high[2][4], low[2][4];
#pragma unroll
                for (int run = 0; run < 2; ++run) two_parts(raw[s][run], unit, high[run], low[run]);
                query[s][0] = intx8{high[0][0], high[0][1], high[0][2], high[0][3], high[1][0], high[1][1], high[1][2], high[1][3]};
                query[s][1] = intx8{low[0][0], low[0][1], low[0][2], low[0][3], low[1][0], low[1][1], low[1][2], low[1][3]};
            }
        }

        // ---- bringing a stage by way of registers: a thread's unit of keys is block `k_block` of key k_key, its values eight `v_eight`
        // of the four tokens from v_key; a wave's lanes also hold the powers of the keys that they multiply.
        const int* table = block_table + static_cast<long>(entry) * max_blocks;
        const long code_bytes = four_bit_codes(page_tokens, kD), power_bytes = four_bit_powers(page_tokens, kD);
        const bool brings = kKeyUnits == kPromptThreads || tid < kKeyUnits;
        const int k_key = 32 * (tid / (32 * kBlocks)) + pass_key(tid & 31), k_block = tid / 32 % kBlocks;
        const int v_key = 4 * (tid / kEights), v_eight = tid % kEights;
        const int p_key = pass_key(j);
        // The pages of a stage.  Loads are the same whatever the stage (what is behind the table reads its last place) and are not
        // waited for before they are used, a stage later.
        struct Pages {
            int k, v, p[2];
        };
        auto entry_of = [&](int key) { return table[min(key >> page_shift, max_blocks - 1)]; };
        auto find = [&](int t) {
            const int key0 = t * kStageKeys;
            Pages at;
            if constexpr (kWide) {
                at.k = at.v = at.p[0] = at.p[1] = entry_of(key0);
            } else {
                at.k = entry_of(key0 + k_key), at.v = entry_of(key0 + v_key);
                at.p[0] = entry_of(key0 + p_key), at.p[1] = entry_of(key0 + 32 + p_key);
            }
            return at;
        };
        auto mapped = [&](int page, int key) { return static_cast<unsigned>(page) < static_cast<unsigned>(pools.pages) && key >> page_shift < max_blocks; };
        // (a page's powers are a sixteenth of its codes)
        const unsigned code_stride = static_cast<unsigned>(code_bytes) * kv_heads;
        const uint8_t* k_codes_base = pools.k_codes + kvh * code_bytes;
        const uint8_t* k_powers_base = pools.k_powers + kvh * power_bytes;
        const uint8_t* v_codes_base = pools.v_codes + kvh * code_bytes;
        const uint8_t* v_powers_base = pools.v_powers + kvh * power_bytes;
        // a lane's own offsets from where the stage's first key, or (pages shorter than a stage) its own key's page begins
        const unsigned k_code_at = four_bit_key(kWide ? k_key : k_key & page_mask, k_block, page_tokens);
        const unsigned v_code_at = four_bit_value(kWide ? v_key : v_key & page_mask, v_eight, kD);
        const unsigned v_power_at = four_bit_value_power(kWide ? v_key : v_key & page_mask, v_eight / 4, kD);
        unsigned k_power_at[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) k_power_at[half] = four_bit_key_power(kWide ? 32 * half + p_key : (32 * half + p_key) & page_mask, 0, kD);
        uint4 k_codes = {0u, 0u, 0u, 0u}, v_codes = {0u, 0u, 0u, 0u};
        unsigned v_powers = 0x7f7f7f7fu;
        unsigned k_powers[2], k_powers_next[2];
        auto fetch = [&](int t, const Pages& at) {
            const int key0 = t * kStageKeys;
            const unsigned token0 = kWide ? key0 & page_mask : 0;            // (pages shorter than a stage: it begins where one does)
            auto place = [&](int page, int key) { return static_cast<unsigned long long>(mapped(page, key) ? page : 0) * code_stride; };
            // of a stage that is not wholly in sight, or has keys without a page, what is not there may be anything: a power of one
            // makes it a number (its keys' scores are masked later)
            if (brings) {
                const int key = key0 + (kWide ? 0 : k_key), v_first = key0 + (kWide ? 0 : v_key);
                const unsigned long long k_place = place(at.k, key), v_place = kWide ? k_place : place(at.v, v_first);
                k_codes = *reinterpret_cast<const uint4*>(k_codes_base + (k_place + 16 * token0) + k_code_at);
                v_codes = *reinterpret_cast<const uint4*>(v_codes_base + (v_place + kD / 2 * token0) + v_code_at);
                v_powers = *reinterpret_cast<const unsigned*>(v_powers_base + (v_place / 16 + kBlocks * token0) + v_power_at);
                const bool k_mapped = mapped(at.k, key), v_mapped = mapped(at.v, v_first);
                if (key0 < group_lo || key0 + kStageKeys > group_hi || !k_mapped || !v_mapped) {
                    if (!k_mapped && key0 + k_key >= group_lo && key0 + k_key < group_hi) unmapped_seen = 1;
                    unsigned hidden = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (key0 + v_key + i < group_lo || key0 + v_key + i >= group_hi || !v_mapped) hidden |= 0xffu << (8 * i);
                    v_powers = (v_powers & ~hidden) | (0x7f7f7f7fu & hidden);
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint8_t* from = k_powers_base + (place(at.p[half], key0 + (kWide ? 0 : 32 * half + p_key)) / 16 + kBlocks * token0) + k_power_at[half];
                if constexpr (kBlocks == 4) k_powers_next[half] = *reinterpret_cast<const unsigned*>(from);
                else k_powers_next[half] = *reinterpret_cast<const unsigned short*>(from);
            }
        };
        // The values on their way into shared memory: by token, two elements at a time, then by element.
        auto deposit = [&](int note, PromptStage<kD>* to) {
            if (brings) {
                to->keys[tid] = k_codes;
                const unsigned clear = ~v_powers;                // a byte of 255 is one of zero here
                unsigned words[4] = {v_codes.x, v_codes.y, v_codes.z, v_codes.w};
                unsigned powers = v_powers;
                if (((clear - 0x01010101u) & v_powers & 0x80808080u) != 0) {
                    unsigned nan_tokens = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) nan_tokens |= (v_powers >> (8 * i) & 255u) == 255u ? 1u << i : 0u;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (nan_tokens >> i & 1u) words[i] = 0, powers = (powers & ~(0xffu << (8 * i))) | (0x7fu << (8 * i));
                    nan_seen[note] = 1;
                    atomicOr(&nan_keys[note][v_eight / 4], static_cast<unsigned long long>(nan_tokens) << v_key);
                }
                float power[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) power[i] = power_of(powers >> (8 * i) & 255u);
                uint2* place = reinterpret_cast<uint2*>(to->values + (v_key / 8) * kD + v_eight) + (v_key / 4 & 1);
                auto pair = [&](auto index) {
                    constexpr int i = decltype(index)::value;
                    unsigned two[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) two[k] = two_bf16<i>(words[k], power[k]);
                    place[2 * (2 * i) * kEights] = uint2{__builtin_amdgcn_perm(two[1], two[0], 0x05040100u), __builtin_amdgcn_perm(two[3], two[2], 0x05040100u)};
                    place[2 * (2 * i + 1) * kEights] = uint2{__builtin_amdgcn_perm(two[1], two[0], 0x07060302u), __builtin_amdgcn_perm(two[3], two[2], 0x07060302u)};
                };
                pair(std::integral_constant<int, 0>{});
                pair(std::integral_constant<int, 1>{});
                pair(std::integral_constant<int, 2>{});
                pair(std::integral_constant<int, 3>{});
            }
        };

        // ---- one pass of a wave: 32 keys against its 32 rows
        auto pass = [&](const PromptStage<kD>* from, const uint4 key[kSteps], int key0, int half, bool full) {
            floatx16 sc;
#pragma unroll
            for (int v = 0; v < 16; ++v) sc[v] = 0.f;
            const int powers = static_cast<int>(k_powers[half] >> (8 * h));
            // Two waves share a SIMD and do best when one multiplies while the other makes weights or unpacks: who is further on in a
            // pass goes first, and what belongs to no pass waits (2,048 rows behind 8,192 tokens 306 us without, 294 with every second 256
            // workgroups ahead, 283 so; whole passes ahead of the rest 285, products ahead of weights 307).
            __builtin_amdgcn_s_setprio(1);
            sc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(low_half(key[0]), query[0][0], sc, 4, 0, 0, powers, 0, power_high);
            sc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(low_half(key[0]), query[0][1], sc, 4, 0, 0, powers, 0, power_low);
            if constexpr (kSteps > 1) {
                sc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(low_half(key[kSteps - 1]), query[kSteps - 1][0], sc, 4, 0, 2, powers, 0, power_high);
                sc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(low_half(key[kSteps - 1]), query[kSteps - 1][1], sc, 4, 0, 2, powers, 0, power_low);
            }
            bf16x8 xv[2][kDT];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt) xv[ks][dt] = __builtin_bit_cast(bf16x8, from->values[(4 * half + 2 * ks + h) * kD + 32 * dt + j]);
            // sc[v]: row j's score of key key0 + 8 h + v (v < 8) or key0 + 16 + 8 h + v - 8
            if (!full) {
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int key_at = key0 + 8 * h + (v & 7) + 16 * (v >> 3);
                    sc[v] = key_at <= row_pos && key_at >= row_lo && key_at >= group_lo && key_at < group_hi ? sc[v] : -INFINITY;
                }
            }
            __builtin_amdgcn_s_setprio(2);
            float top = sc[0];
#pragma unroll
            for (int v = 1; v < 16; ++v) top = fmaxf(top, sc[v]);
            top *= to_log2;
            if (__any(top > m_ref + kRaise)) {                   // -inf + 8 is -inf: the first scores always raise
                const float m_new = fmaxf(m_ref, ceilf(max_lanes<32>(top)));
                const float keep = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_ref - m_new);
                m_ref = m_new;
                l_run *= keep;
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                    for (int v = 0; v < 16; ++v) acc[dt][v] *= keep;
            }
            const float shift = m_ref == -INFINITY ? 0.f : -m_ref;
            bf16x8 pt[2];
#pragma unroll
            for (int v = 0; v < 16; ++v) pt[v >> 3][v & 7] = static_cast<__bf16>(__builtin_amdgcn_exp2f(fmaf(sc[v], to_log2, shift)));
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const uint4 packed = __builtin_bit_cast(uint4, pt[ks]);
                const unsigned pairs[4] = {packed.x, packed.y, packed.z, packed.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    l_run = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pairs[i]), __builtin_bit_cast(bf16x2, 0x3f803f80u), l_run, false);
            }
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xv[ks][dt], pt[ks], acc[dt], 0, 0, 0);
            __builtin_amdgcn_s_setprio(0);
        };
        // Which of a block's elements register v of tile dt holds: row r = 8 (v / 4) + 4 h + v % 4 of the tile is place 32 dt + r.
        auto block_of = [&](int dt, int v) {
            const int at = 32 * dt + 8 * (v / 4) + 4 * h + v % 4;
            return (at % kEights) / 4;
        };
        auto spoil = [&](int t, int note) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const unsigned long long keys = nan_keys[note][b];
                if (keys == 0) continue;                         // (the same for the workgroup)
                const int first = max(row_lo - t * kStageKeys, 0), last = min(row_pos - t * kStageKeys, kStageKeys - 1);
                unsigned long long seen = last >= first ? (~0ull >> (63 - last + first)) << first : 0ull;
                if ((seen & keys) != 0) {
#pragma unroll
                    for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                        for (int v = 0; v < 16; ++v)
                            if (block_of(dt, v) == b) acc[dt][v] = __builtin_nanf("");
                }
            }
        };

        const int t_begin = group_lo / kStageKeys, t_end = (group_hi + kStageKeys - 1) / kStageKeys;
        // stages of which every row of the wave sees every key
        const int plain_begin = (max(full_lo, group_lo) + kStageKeys - 1) / kStageKeys, plain_end = min(full_hi, group_hi) / kStageKeys;
        // Stage t + 1 is brought to shared memory in the middle of round t, from registers that were asked for a round before: the
        // instructions that unpack it go beside the first half's second product.  (Every round asks for a stage, the last one again
        // where there is no further: see `find`.)
        fetch(t_begin, find(t_begin));
        Pages ahead = find(min(t_begin + 1, t_end - 1));
        deposit(0, &stages[0]);
        unsigned k_powers_ready[2] = {k_powers_next[0], k_powers_next[1]};
        k_powers[0] = k_powers_next[0], k_powers[1] = k_powers_next[1];
        fetch(min(t_begin + 1, t_end - 1), ahead);
        ahead = find(min(t_begin + 2, t_end - 1));
        shared_barrier();
        // `note`, `next_note`, `old_note`: whose NaN keys are read, written and cleared while stage t is worked on
        auto round = [&](const PromptStage<kD>* __restrict__ reading, PromptStage<kD>* __restrict__ writing, int t, int note, int next_note, int old_note) {
            const int any_nan = nan_seen[note];                   // (asked for with the keys, used behind them)
            uint4 keys[2][kSteps];                               // (of both passes: the second does not wait for its own)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int s = 0; s < kSteps; ++s) keys[half][s] = reading->keys[(half * kBlocks + 2 * s + h) * 32 + j];
            const bool plain = t >= plain_begin && t < plain_end;    // nothing to mask: most stages of a long context
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int key0 = t * kStageKeys + half * kPassKeys;
                if (plain || (key0 < key_hi && key0 + kPassKeys > key_lo)) pass(reading, keys[half], key0, half, plain);
                if (half == 0) {
                    if (t + 1 < t_end) deposit(next_note, writing);
                    k_powers_ready[0] = k_powers_next[0], k_powers_ready[1] = k_powers_next[1];
                    fetch(min(t + 2, t_end - 1), ahead);
                    ahead = find(min(t + 3, t_end - 1));
                }
            }
            if (any_nan != 0) spoil(t, note);
            if (tid < kBlocks) nan_keys[old_note][tid] = 0;
            if (tid == 0) nan_seen[old_note] = 0;
        };
        int note = 0;
        for (int t = t_begin; t < t_end; ++t) {
            const int cur = (t - t_begin) & 1, next_note = note == 2 ? 0 : note + 1, old_note = note == 0 ? 2 : note - 1;
            round(&stages[cur], &stages[cur ^ 1], t, note, next_note, old_note);
            note = next_note;
            k_powers[0] = k_powers_ready[0], k_powers[1] = k_powers_ready[1];
            shared_barrier();
        }
    }
    __syncthreads();
    const bool poisoned = unmapped_seen != 0;
    if (!row_ok) return;
    float l_row = add_lanes<32>(l_run);
    if (poisoned && row_pos >= 0) l_row = __builtin_nanf("");
    if (l_row != l_row) m_ref = fmaxf(m_ref, 0.f);               // (a result of NaN counts, whatever its maximum)
    const bool nothing = m_ref == -INFINITY;
    const long row_head = static_cast<long>(tile_row0 + j) * q_heads + head, slot = row_head * splits + blockIdx.y;
    if (splits > 1) {
        if (h == 0) part_ml[2 * slot] = m_ref, part_ml[2 * slot + 1] = l_row;
        if (nothing) return;
    }
    const float inv = nothing ? 0.f : 1.f / l_row;
    // Places that differ by a whole row of eights are neighbouring elements: registers of the same place % kEights, in the order of the
    // places, are the eight elements of one eight.
#pragma unroll
    for (int e = 0; e < kEights / 2; ++e) {
        const int at0 = 8 * (e / 4) + e % 4;                      // its place, 4 h aside
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int at = at0 + i * kEights, dt = at / 32, r = at % 32;
            x[i] = acc[dt][4 * (r / 8) + r % 4];
        }
        if (splits > 1) {
            floatx4* to = reinterpret_cast<floatx4*>(part_acc + slot * kD + 8 * (at0 + 4 * h));
            to[0] = floatx4{x[0], x[1], x[2], x[3]}, to[1] = floatx4{x[4], x[5], x[6], x[7]};
        } else {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = bf16_bits_from_float(x[2 * i] * inv) | static_cast<unsigned>(bf16_bits_from_float(x[2 * i + 1] * inv)) << 16;
            *reinterpret_cast<uint4*>(out + row_head * kD + 8 * (at0 + 4 * h)) = uint4{w[0], w[1], w[2], w[3]};
        }
    }
}

}  // namespace leone

using namespace leone;

extern "C" int leone_four_bit_prefill(const void* q, void* out, const void* k_codes, const void* k_powers, const void* v_codes, const void* v_powers,
                                      int pages, const int* positions, const int* tiles, int n_groups, int rows, const int* block_table, int max_blocks,
                                      int entries, int q_heads, int kv_heads, int head_dim, int page_tokens, float scale, int window, int splits,
                                      float* part_acc, float* part_ml, hipStream_t stream) {
    const char* what = "four_bit_prefill";
    const FourBitPools pools = read_pools(k_codes, k_powers, v_codes, v_powers, pages);
    if (check_four_bit(what, pools, kv_heads, head_dim, page_tokens, max_blocks)) return 1;
    LEONE_REQUIRE(q && out && positions && tiles && block_table, "%s: null pointer", what);
    LEONE_REQUIRE(head_dim == 64 || head_dim == 128, "%s: heads of 64 or 128 elements, not %d", what, head_dim);
    LEONE_REQUIRE(page_tokens >= 16 && (page_tokens & (page_tokens - 1)) == 0, "%s: pages of a power of two tokens from 16 on, not %d", what, page_tokens);
    LEONE_REQUIRE(scale > 0.f, "%s: the score scale must be positive", what);
    LEONE_REQUIRE(rows > 0, "%s: %d rows", what, rows);
    LEONE_REQUIRE(n_groups > 0 && entries > 0 && q_heads > 0 && q_heads % kv_heads == 0, "%s: %d tile groups, %d entries, %d query heads over %d kv heads",
                  what, n_groups, entries, q_heads, kv_heads);
    LEONE_REQUIRE(static_cast<long>(n_groups) * q_heads <= 0x7fffffffL / kTileRows, "%s: too many tile groups", what);
    LEONE_REQUIRE(window >= 0 && splits >= 1 && splits <= kMaxRanges, "%s: window %d must not be negative, splits %d in 1..%d", what, window, splits,
                  kMaxRanges);
    LEONE_REQUIRE(splits == 1 || (part_acc && part_ml && reinterpret_cast<uintptr_t>(part_acc) % 16 == 0), "%s: %d ranges need the workspace", what, splits);
    LEONE_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) % 16 == 0, "%s: queries and results start at multiples of 16 bytes", what);
    LEONE_REQUIRE(four_bit_codes(page_tokens, head_dim) * kv_heads < 0x7fffffffL, "%s: a page of %d heads is too large", what, kv_heads);
    int page_shift = 0;
    while ((1 << page_shift) < page_tokens) ++page_shift;
    const dim3 grid(n_groups * q_heads, splits);
#define LEONE_PREFILL_CALL(D, WIDE)                                                                                                            \
    four_bit_prefill_kernel<D, WIDE><<<grid, kPromptThreads, 0, stream>>>(static_cast<const bf16_t*>(q), static_cast<bf16_t*>(out), pools,     \
                                                                          positions, tiles, n_groups, rows, block_table, max_blocks, entries, q_heads, \
                                                                          kv_heads, page_shift, scale * kLog2e, window, splits, part_acc, part_ml)
#define LEONE_PREFILL(D)                                             \
    do {                                                             \
        if (page_tokens >= kStageKeys) LEONE_PREFILL_CALL(D, true);  \
        else LEONE_PREFILL_CALL(D, false);                           \
    } while (0)
    if (head_dim == 64) LEONE_PREFILL(64);
    else LEONE_PREFILL(128);
#undef LEONE_PREFILL
#undef LEONE_PREFILL_CALL
    LEONE_LAUNCH_CHECK(what);
    if (splits > 1) {
        merge_four_bit_shares(part_acc, part_ml, out, kBF16, static_cast<long>(n_groups) * kPromptWaves * kTileRows, q_heads, head_dim, splits, tiles, rows, stream);
        LEONE_LAUNCH_CHECK("four_bit_merge");
    }
    return 0;
}
