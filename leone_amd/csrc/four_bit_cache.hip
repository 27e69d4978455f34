// What fills the cache of 4 bits an element (four_bit.h) and what reads it back as values.
//
// Filling it: a row of the fused q/k/v projection becomes query heads (RMS norm of the head times a gain, rotation; rounded once, to
// the engine's type) and cached keys and values.  A key is normed and rotated in 64 bits and stays there up to its codes: which
// of two neighbouring codes an element gets is decided by a comparison, and one that lies next to the border between
// them falls on its own side whatever order the squares were added in.  Values are only scaled by a power of two, which float does
// exactly.
//
// A lane has eight neighbouring elements, a head dim / 8 lanes (rounded up to a power of two), a wave as many rows of one
// head as fit: four rows of 128.  So a wave's keys of a block and its values of eight elements are neighbouring bytes of the cache
// where its rows are neighbouring tokens, and the four lanes of a block find its largest element by two exchanges.
//
// Few rows wait for trips to memory one behind the other, so everything that needs no other load is asked for at once (one row of 32 heads
// over 8: 3.6 us with the launch, 6.1 where a load was converted before the next was sent).  Many rows wait for instructions and memory in
// turn: 2,048 rows 18.4 us, 44 MB, of which the 64-bit arithmetic of the keys is 3.9 and the rotation 3 (float keys, no rotation and
// no norms 10.1); four heads a wave, which share a row's angles, were level.
#include "common.h"
#include "four_bit.h"
#include "leone_hip.h"

#include <math.h>

namespace leone {

constexpr int kFillThreads = 256;

struct FillShape {
    int rows, q_heads, kv_heads, dim, page_tokens, max_blocks, entries;
    int page_shift;              // of pages of a power of two tokens, else -1
    int kv_written;              // key and value heads that are written: all or none
    long row_width;              // elements from row to row
    int planes;
    long plane;
    float eps;
    const float* cos_table;      // [table_positions, rotary_half], null: no rotation
    const float* sin_table;
    int table_positions, rotary_half, pairing;
};

// Eight neighbouring elements as they were loaded, unpacked where they are used: what a row starts from is asked for at once, and
// nothing waits for one before the next is asked for.
template <typename TIn>
struct Raw {
    uint4 v[sizeof(TIn) / 2];
    __device__ void load(const TIn* from) {
#pragma unroll
        for (unsigned i = 0; i < sizeof(TIn) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(from)[i];
    }
    template <typename Acc>
    __device__ void get(Acc x[8]) const {
        const unsigned w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
        if constexpr (sizeof(TIn) == 4) {
            const unsigned u[4] = {v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]), x[4 + i] = __uint_as_float(u[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};
// The planes of a product cut along K added up in order, the first of them as it was loaded.
template <typename TIn, typename Acc>
__device__ inline void add_planes(const Raw<TIn>& first, const TIn* __restrict__ from, int planes, long plane, Acc out[8]) {
    first.get(out);
    for (int p = 1; p < planes; ++p) {
        Raw<TIn> next;
        float part[8];
        next.load(from + p * plane);
        next.get(part);
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] += static_cast<Acc>(part[i]);
    }
}
// What a lane starts from beside its own elements: its gains, and (kWholeHalves) its angles.
struct Beside {
    uint4 gain[2];
    float4 cosine[2], sine[2];
    __device__ void gains(int dtype, float g[8]) const {
        if (dtype == kF32) Raw<float>{{gain[0], gain[1]}}.get(g);
        else Raw<bf16_t>{{gain[0]}}.get(g);
    }
};

__device__ inline float root(float v) { return sqrtf(v); }
__device__ inline double root(double v) { return sqrt(v); }

// The value that the lane kOff further (or nearer) holds; every lane of the wave takes part.
template <int kOff, typename T>
__device__ inline T of_partner(T v, int lane) {
    const Pair<T> both = lane_pair<kOff>(v);
    if constexpr (kOff >= 16) return lane & kOff ? both.a : both.b;
    else return both.b;
}

// How a head is rotated: not at all, whole in halves (dim a power of two: the partners are half a head's lanes away, the angles are read
// in runs), or in any other way (partners are loaded a second time, angles one by one).
enum Turn : int { kNoTurn = 0, kWholeHalves = 1, kAnyTurn = 2 };

// Eight elements of a query or key head: normed and rotated.  `at` is the lane's first element; lanes behind the head (at >= dim)
// take part in the sum with nothing.
template <int kSpan, int kTurn, typename TIn, typename Acc>
__device__ inline void make_eight(const Raw<TIn>& raw, const Beside& beside, const TIn* __restrict__ head, int at, int lane, const FillShape& s,
                                  const AnyVec& gain, int pos, Acc x[8]) {
    const bool in_head = at < s.dim;
    const int half = s.rotary_half;
    const long angles = static_cast<long>(max(pos < s.table_positions ? pos : s.table_positions - 1, 0)) * half;   // (the host checks the bound)
    add_planes<TIn, Acc>(raw, head + at, in_head ? s.planes : 1, s.plane, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = in_head ? x[i] : 0;
    // the partners, where they are not among the lane's own
    const bool turned = kTurn == kAnyTurn && at < 2 * half;
    const bool apart = turned && s.pairing == 0;
    [[maybe_unused]] Acc other[8];
    auto partner = [&](int d) { return d < half ? d + half : d - half; };
    if constexpr (kTurn == kAnyTurn) {
#pragma unroll
        for (int i = 0; i < 8; ++i) other[i] = 0;
        if (apart && in_head) {
            if (half % 8 == 0) {
                Raw<TIn> theirs;
                theirs.load(head + partner(at));
                add_planes<TIn, Acc>(theirs, head + partner(at), s.planes, s.plane, other);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at + i < 2 * half)
                        for (int p = 0; p < s.planes; ++p) {
                            const TIn v = head[p * s.plane + partner(at + i)];
                            other[i] += static_cast<Acc>(to_float(v));
                        }
            }
        }
    }
    if (gain.ptr) {
        Acc squares = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) squares += x[i] * x[i];
        squares = join_span<kSpan>(squares, [](Acc a, Acc b) { return a + b; });
        const Acc inv = Acc(1) / root(squares / static_cast<Acc>(s.dim) + static_cast<Acc>(s.eps));
        float g[8];
        beside.gains(gain.dtype, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * static_cast<Acc>(g[i]) * inv;
        if (in_head) {
            if (apart) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (at + i < 2 * half) other[i] = other[i] * static_cast<Acc>(load_any(gain, partner(at + i))) * inv;
            }
        }
    }
    if constexpr (kTurn == kWholeHalves) {
        const bool first = (lane & (kSpan / 2)) == 0;
        const float c[8] = {beside.cosine[0].x, beside.cosine[0].y, beside.cosine[0].z, beside.cosine[0].w,
                            beside.cosine[1].x, beside.cosine[1].y, beside.cosine[1].z, beside.cosine[1].w};
        const float n[8] = {beside.sine[0].x, beside.sine[0].y, beside.sine[0].z, beside.sine[0].w,
                            beside.sine[1].x, beside.sine[1].y, beside.sine[1].z, beside.sine[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const Acc o = of_partner<kSpan / 2>(x[i], lane), cosine = c[i], sine = first ? -n[i] : n[i];
            x[i] = x[i] * cosine + o * sine;
        }
    }
    if (!turned) return;
    if (s.pairing != 0) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if (at + i >= 2 * half) continue;
            const Acc cosine = s.cos_table[angles + (at + i) / 2], sine = s.sin_table[angles + (at + i) / 2];
            const Acc a = x[i], b = x[i + 1];
            x[i] = a * cosine - b * sine;
            x[i + 1] = a * sine + b * cosine;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int d = at + i;
        if (d >= 2 * half) continue;
        const bool first = d < half;
        const Acc cosine = s.cos_table[angles + (first ? d : d - half)], sine = s.sin_table[angles + (first ? d : d - half)];
        x[i] = first ? x[i] * cosine - other[i] * sine : other[i] * sine + x[i] * cosine;
    }
}

// The power of a block of 32 (four neighbouring lanes) and the lane's eight codes.
__device__ inline unsigned long long magnitude(double v) { return __builtin_bit_cast(unsigned long long, v) & 0x7fffffffffffffffull; }
__device__ inline unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }
__device__ inline int block_power(unsigned long long top) {
    const int exponent = static_cast<int>(top >> 52);
    if (exponent == 0x7ff) return kNanPower;
    const int power = exponent - 1023 - ((top & 0xfffffffffffffull) > 0xc000000000000ull ? 1 : 2);       // above 1.75 times a power of two?
    return min(max(power, -126), 127) + 127;
}
__device__ inline int block_power(unsigned top) {
    const int exponent = static_cast<int>(top >> 23);
    if (exponent == 0xff) return kNanPower;
    const int power = exponent - 127 - ((top & 0x7fffffu) > 0x600000u ? 1 : 2);
    return max(power, -126) + 127;
}
// x / 2^(power - 127) as a float that rounds to the same code: of a 64-bit number the float towards zero, its last bit set where
// something was cut off.
__device__ inline float in_units(double x, int power) {
    const double y = x * __builtin_bit_cast(double, static_cast<unsigned long long>(1023 + 127 - power) << 52);
    const float f = static_cast<float>(y);
    const double back = f;
    unsigned bits = __builtin_bit_cast(unsigned, f);
    if (back != y) bits = (fabs(back) > fabs(y) ? bits - 1 : bits) | 1u;
    return __builtin_bit_cast(float, bits);
}
__device__ inline float in_units(float x, int power) { return ldexpf(x, 127 - power); }

template <typename Acc>
__device__ inline unsigned eight_codes(const Acc x[8], int& power) {
    decltype(magnitude(Acc())) top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude(x[i]));
    top = join_span<4>(top, [](auto a, auto b) { return a > b ? a : b; });
    power = block_power(top);
    const int by = power == kNanPower ? 127 : power;
    unsigned codes = 0;
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, in_units(x[0], by), in_units(x[1], by), 1.0f, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, in_units(x[2], by), in_units(x[3], by), 1.0f, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, in_units(x[4], by), in_units(x[5], by), 1.0f, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, in_units(x[6], by), in_units(x[7], by), 1.0f, 3);
    return codes;
}

template <int kSpan, int kTurn, typename TIn, typename T>
__global__ void __launch_bounds__(kFillThreads)
four_bit_fill_kernel(const TIn* __restrict__ qkv, T* __restrict__ q_out, FourBitPools pools, AnyVec q_gain, AnyVec k_gain,
                     const int* __restrict__ positions, const int* __restrict__ row_entry, const int* __restrict__ block_table, FillShape s) {
    constexpr int kRows = kWave / kSpan;                          // rows of one head a wave takes
    const int lane = threadIdx.x % kWave;
    const int head = blockIdx.x * (kFillThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int row_run = blockIdx.y;
    if (head >= s.q_heads + s.kv_written) return;
    const int row = row_run * kRows + lane / kSpan;
    const int at = lane % kSpan * 8;
    const bool exists = row < s.rows;
    const int from_row = exists ? row : s.rows - 1;               // (every lane takes part in the exchanges)
    const bool is_query = head < s.q_heads, is_key = !is_query && head < s.q_heads + s.kv_heads;
    const TIn* from = qkv + static_cast<long>(from_row) * s.row_width + static_cast<long>(head) * s.dim;
    const int pos = positions[from_row], entry = row_entry[from_row];
    const int read_at = min(at, s.dim - 8);                       // (lanes behind the head read its last eight and drop them)
    Raw<TIn> raw;
    raw.load(from + read_at);
    const AnyVec gain = is_query ? q_gain : k_gain;
    Beside beside;
    if (gain.ptr != nullptr && (is_query || is_key)) {
        if (gain.dtype == kF32) {
            const uint4* g = reinterpret_cast<const uint4*>(static_cast<const float*>(gain.ptr) + read_at);
            beside.gain[0] = g[0], beside.gain[1] = g[1];
        } else {
            beside.gain[0] = *reinterpret_cast<const uint4*>(static_cast<const bf16_t*>(gain.ptr) + read_at);
        }
    }
    if constexpr (kTurn == kWholeHalves) {
        if (is_query || is_key) {
            const long angles = static_cast<long>(max(pos < s.table_positions ? pos : s.table_positions - 1, 0)) * s.rotary_half + (at & (s.rotary_half - 1));
            const float4* c = reinterpret_cast<const float4*>(s.cos_table + angles);
            const float4* n = reinterpret_cast<const float4*>(s.sin_table + angles);
            beside.cosine[0] = c[0], beside.cosine[1] = c[1], beside.sine[0] = n[0], beside.sine[1] = n[1];
        }
    }
    if (is_query) {
        float x[8];
        make_eight<kSpan, kTurn, TIn, float>(raw, beside, from, at, lane, s, q_gain, pos, x);
        if (!exists || at >= s.dim) return;
        T* to = q_out + (static_cast<long>(row) * s.q_heads + head) * s.dim + at;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(to) = float4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<float4*>(to + 4) = float4{x[4], x[5], x[6], x[7]};
        } else {
            unsigned w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = bf16_bits_from_float(x[2 * i]) | static_cast<unsigned>(bf16_bits_from_float(x[2 * i + 1])) << 16;
            *reinterpret_cast<uint4*>(to) = uint4{w[0], w[1], w[2], w[3]};
        }
        return;
    }
    const int kvh = head - s.q_heads - (is_key ? 0 : s.kv_heads);
    // where the row goes is looked up while its numbers are made
    const bool placed = exists && at < s.dim && pos >= 0 && entry >= 0 && entry < s.entries;
    const int block = s.page_shift >= 0 ? pos >> s.page_shift : pos / s.page_tokens, token = pos - block * s.page_tokens;
    const int page = placed ? mapped_page(block_table + static_cast<long>(entry) * s.max_blocks, block, s.max_blocks, pools.pages) : -1;
    int power;
    unsigned codes;
    if (is_key) {
        double x[8];
        make_eight<kSpan, kTurn, TIn, double>(raw, beside, from, at, lane, s, k_gain, pos, x);
        codes = eight_codes(x, power);
    } else if (s.planes == 1) {
        float x[8];
        raw.get(x);
        codes = eight_codes(x, power);
    } else {
        double x[8];
        add_planes<TIn, double>(raw, from + read_at, s.planes, s.plane, x);
        codes = eight_codes(x, power);
    }
    if (page < 0) return;                                         // the host reserves the pages before the launch
    const long place = static_cast<long>(page) * s.kv_heads + kvh;
    const long code_base = place * four_bit_codes(s.page_tokens, s.dim), power_base = place * four_bit_powers(s.page_tokens, s.dim);
    if (is_key) {
        *reinterpret_cast<unsigned*>(pools.k_codes + code_base + four_bit_key(token, at / kBlock, s.page_tokens) + at % kBlock / 2) = codes;
        if (at % kBlock == 0) pools.k_powers[power_base + four_bit_key_power(token, at / kBlock, s.dim)] = static_cast<uint8_t>(power);
    } else {
        *reinterpret_cast<unsigned*>(pools.v_codes + code_base + four_bit_value(token, at / 8, s.dim)) = codes;
        if (at % kBlock == 0) pools.v_powers[power_base + four_bit_value_power(token, at / kBlock, s.dim)] = static_cast<uint8_t>(power);
    }
}

// Reading rows back: a thread has eight elements of a key or a value.  A number of two bits times a power of two is a bfloat16
// as it is.  Rows without a page give NaN.
__global__ void __launch_bounds__(kFillThreads)
four_bit_rows_kernel(FourBitPools pools, const int* __restrict__ positions, const int* __restrict__ row_entry, const int* __restrict__ block_table,
                     int max_blocks, int entries, bf16_t* __restrict__ k_out, bf16_t* __restrict__ v_out, long items, int kv_heads, int dim,
                     int page_tokens) {
    const long item = static_cast<long>(blockIdx.x) * kFillThreads + threadIdx.x;
    if (item >= items) return;
    const int eights = dim / 8;
    const long head_row = item / eights;
    const int eight = static_cast<int>(item - head_row * eights);
    const int row = static_cast<int>(head_row / kv_heads), kvh = static_cast<int>(head_row - static_cast<long>(row) * kv_heads);
    const int pos = positions[row], entry = row_entry[row];
    int page = -1;
    const int block = pos / page_tokens, token = pos - block * page_tokens;
    if (pos >= 0 && entry >= 0 && entry < entries) page = mapped_page(block_table + static_cast<long>(entry) * max_blocks, block, max_blocks, pools.pages);
    uint4 k = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu}, v = k;
    if (page >= 0) {
        const long place = static_cast<long>(page) * kv_heads + kvh;
        const long code_base = place * four_bit_codes(page_tokens, dim), power_base = place * four_bit_powers(page_tokens, dim);
        const unsigned k_codes = *reinterpret_cast<const unsigned*>(pools.k_codes + code_base + four_bit_key(token, eight / 4, page_tokens) + eight % 4 * 4);
        const unsigned v_codes = *reinterpret_cast<const unsigned*>(pools.v_codes + code_base + four_bit_value(token, eight, dim));
        const float kp = power_of(pools.k_powers[power_base + four_bit_key_power(token, eight / 4, dim)]);
        const float vp = power_of(pools.v_powers[power_base + four_bit_value_power(token, eight / 4, dim)]);
        k = uint4{two_bf16<0>(k_codes, kp), two_bf16<1>(k_codes, kp), two_bf16<2>(k_codes, kp), two_bf16<3>(k_codes, kp)};
        v = uint4{two_bf16<0>(v_codes, vp), two_bf16<1>(v_codes, vp), two_bf16<2>(v_codes, vp), two_bf16<3>(v_codes, vp)};
    }
    const long to = head_row * dim + eight * 8;
    *reinterpret_cast<uint4*>(k_out + to) = k;
    *reinterpret_cast<uint4*>(v_out + to) = v;
}

template <int kSpan, typename TIn, typename T>
static void launch_fill_span(const void* qkv, void* q_out, const FourBitPools& pools, AnyVec q_gain, AnyVec k_gain, const int* positions,
                             const int* row_entry, const int* block_table, const FillShape& s, int turn, hipStream_t stream) {
    const dim3 blocks(ceil_div(s.q_heads + s.kv_written, kFillThreads / kWave), ceil_div(s.rows, kWave / kSpan));
#define LEONE_FILL(TURN)                                                                                                                  \
    case TURN:                                                                                                                            \
        four_bit_fill_kernel<kSpan, TURN, TIn, T><<<blocks, kFillThreads, 0, stream>>>(                                                   \
            static_cast<const TIn*>(qkv), static_cast<T*>(q_out), pools, q_gain, k_gain, positions, row_entry, block_table, s);           \
        break;
    switch (turn) { LEONE_FILL(kNoTurn) LEONE_FILL(kWholeHalves) LEONE_FILL(kAnyTurn) }
#undef LEONE_FILL
}

template <typename TIn, typename T>
static void launch_fill(const void* qkv, void* q_out, const FourBitPools& pools, AnyVec q_gain, AnyVec k_gain, const int* positions,
                        const int* row_entry, const int* block_table, const FillShape& s, hipStream_t stream) {
    const int span = s.dim <= 32 ? 4 : s.dim <= 64 ? 8 : s.dim <= 128 ? 16 : 32;
    const bool aligned = (reinterpret_cast<uintptr_t>(s.cos_table) | reinterpret_cast<uintptr_t>(s.sin_table)) % 16 == 0;
    const int turn = s.cos_table == nullptr ? kNoTurn
                     : s.pairing == 0 && 2 * s.rotary_half == s.dim && s.dim == 8 * span && aligned ? kWholeHalves : kAnyTurn;
#define LEONE_SPAN(SPAN)                                                                                                                       \
    case SPAN: launch_fill_span<SPAN, TIn, T>(qkv, q_out, pools, q_gain, k_gain, positions, row_entry, block_table, s, turn, stream); break;
    switch (span) { LEONE_SPAN(4) LEONE_SPAN(8) LEONE_SPAN(16) LEONE_SPAN(32) }
#undef LEONE_SPAN
}

}  // namespace leone

using namespace leone;

extern "C" int leone_four_bit_fill(const void* qkv, int qkv_dtype, int qkv_planes, long qkv_plane, long row_width, void* q_out, int dtype,
                                   void* k_codes, void* k_powers, void* v_codes, void* v_powers, int pages, const void* q_gain,
                                   const void* k_gain, int gain_dtype, float eps, const float* cos_table, const float* sin_table,
                                   int table_positions, int rotary_dim, int pairing, const int* positions, const int* row_entry,
                                   const int* block_table, int max_blocks, int entries, int rows, int q_heads, int kv_heads, int head_dim,
                                   int page_tokens, int write_cache, hipStream_t stream) {
    const char* what = "four_bit_fill";
    const FourBitPools pools{static_cast<uint8_t*>(k_codes), static_cast<uint8_t*>(k_powers), static_cast<uint8_t*>(v_codes),
                             static_cast<uint8_t*>(v_powers), pages};
    if (check_four_bit(what, pools, kv_heads, head_dim, page_tokens, max_blocks)) return 1;
    LEONE_REQUIRE(qkv && q_out && positions && row_entry && block_table, "%s: null pointer", what);
    LEONE_REQUIRE((dtype == kF32 || dtype == kBF16) && (qkv_dtype == dtype || qkv_dtype == kF32), "%s: the input is of the queries' type or float32", what);
    LEONE_REQUIRE(gain_dtype == kF32 || gain_dtype == kBF16, "%s: unknown type of the gains", what);
    LEONE_REQUIRE(rows > 0 && q_heads > 0 && entries > 0, "%s: rows %d, query heads %d, entries %d must be positive", what, rows, q_heads, entries);
    LEONE_REQUIRE(qkv_planes >= 1 && qkv_planes <= 64 && (qkv_planes == 1 || qkv_plane % 8 == 0), "%s: %d planes of input", what, qkv_planes);
    const long width = (static_cast<long>(q_heads) + 2L * kv_heads) * head_dim;
    LEONE_REQUIRE(row_width >= width && row_width % 8 == 0, "%s: rows of %ld elements for heads of %ld", what, row_width, width);
    LEONE_REQUIRE((q_gain == nullptr) == (k_gain == nullptr), "%s: q and k gains come together", what);
    LEONE_REQUIRE((cos_table == nullptr) == (sin_table == nullptr), "%s: cos and sin tables come together", what);
    LEONE_REQUIRE(!cos_table || (table_positions > 0 && rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim),
                  "%s: tables of %d positions for a rotation of %d of %d elements", what, table_positions, rotary_dim, head_dim);
    LEONE_REQUIRE(pairing == 0 || pairing == 1, "%s: unknown pairing %d", what, pairing);
    LEONE_REQUIRE((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(q_gain) |
                   reinterpret_cast<uintptr_t>(k_gain)) % 16 == 0, "%s: the projection, the queries and the gains start at multiples of 16 bytes", what);
    LEONE_REQUIRE(rows <= 2 * 65535, "%s: too many rows for one launch", what);     // (two of 256 elements are the fewest a wave takes)
    const int page_shift = (page_tokens & (page_tokens - 1)) == 0 ? __builtin_ctz(page_tokens) : -1;
    const FillShape s{rows, q_heads, kv_heads, head_dim, page_tokens, max_blocks, entries, page_shift, write_cache ? 2 * kv_heads : 0, row_width, qkv_planes, qkv_plane, eps, cos_table,
                      sin_table, table_positions, cos_table ? rotary_dim / 2 : 0, pairing};
    const AnyVec qg{q_gain, gain_dtype}, kg{k_gain, gain_dtype};
    if (dtype == kF32) launch_fill<float, float>(qkv, q_out, pools, qg, kg, positions, row_entry, block_table, s, stream);
    else if (qkv_dtype == kF32) launch_fill<float, bf16_t>(qkv, q_out, pools, qg, kg, positions, row_entry, block_table, s, stream);
    else launch_fill<bf16_t, bf16_t>(qkv, q_out, pools, qg, kg, positions, row_entry, block_table, s, stream);
    LEONE_LAUNCH_CHECK(what);
    return 0;
}

extern "C" int leone_four_bit_rows(const void* k_codes, const void* k_powers, const void* v_codes, const void* v_powers, int pages,
                                   const int* positions, const int* row_entry, const int* block_table, int max_blocks, int entries,
                                   void* k_out, void* v_out, int rows, int kv_heads, int head_dim, int page_tokens, hipStream_t stream) {
    const char* what = "four_bit_rows";
    auto bytes = [](const void* p) { return const_cast<uint8_t*>(static_cast<const uint8_t*>(p)); };
    const FourBitPools pools{bytes(k_codes), bytes(k_powers), bytes(v_codes), bytes(v_powers), pages};
    if (check_four_bit(what, pools, kv_heads, head_dim, page_tokens, max_blocks)) return 1;
    LEONE_REQUIRE(positions && row_entry && block_table && k_out && v_out, "%s: null pointer", what);
    LEONE_REQUIRE(rows > 0 && entries > 0, "%s: rows %d and entries %d must be positive", what, rows, entries);
    LEONE_REQUIRE((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16 == 0, "%s: the results start at multiples of 16 bytes", what);
    const long items = static_cast<long>(rows) * kv_heads * (head_dim / 8);
    LEONE_REQUIRE(items < 0x7fffffffL * kFillThreads, "%s: too many rows for one launch", what);
    four_bit_rows_kernel<<<ceil_div(items, kFillThreads), kFillThreads, 0, stream>>>(
        pools, positions, row_entry, block_table, max_blocks, entries, static_cast<bf16_t*>(k_out), static_cast<bf16_t*>(v_out), items, kv_heads,
        head_dim, page_tokens);
    LEONE_LAUNCH_CHECK(what);
    return 0;
}
