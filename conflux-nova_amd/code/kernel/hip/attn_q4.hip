// attn_q4.hip -- attention over the 4-bit pages (kv_q4.h): one query token per session
// (decode), or a ragged chunk of new tokens per session, causally.
//
// o_h = sum_t softmax_t(q_h . k_t / sqrt(HD)) v_t, k_t and v_t the values that the codes
// and their powers of two stand for, over keys [0, n_keys) or, for row r of a chunk,
// [0, n_past + r].
//
// Numbers.  K goes into the block-scaled matrix instructions as the page holds it.  The
// query goes in as five 6-bit terms (steps of 1/8 up to 2, each 2^-5 of the one before,
// with a power of two per 32 dims): it is held to 2^-24 of the largest of its 32 dims, and
// sums are fp32.  V's values have one bit of mantissa, so a tile of 64 keys whose powers of two
// lie close together (a window of eight, kSpread) is exact in fp16, and a weight goes in as
// two fp16 terms, to 2^-22 of itself or, where fp16 ends first, to 2^-24.  The largest weight
// of that row in the tile stands at 2^kLow or more, so 2^-24 is 2^-26 of that weight.  Any other
// tile (powers far apart, blocks of zeros, NaN, values past fp16's normal numbers) takes V as bf16 with its
// power of two, exact too, and a weight as the exact sum of three bf16 terms (8 bits each).
// Sums are fp32.
//
// One pass over the keys with a running reference and sum of the softmax.  The reference
// m of the weights 2^(s - m) follows the largest score of the tiles, both ways and
// lazily: a tile's largest weight may lie from 2^kLow to 2^kHigh before the sums are rescaled.  It
// goes down no further than kDrop below its highest, so that the sums stay inside fp32: a
// tile further down, whose largest weight may be anything, loses 2^-104 of the row's largest
// per key (2^-24 of a unit that is 2^-kDrop of it).
//
// What bounds it (one MI355X).  Few columns: HBM where the keys are many (8 x 32768 keys, 14B, 285
// MB: 51 us, 5.6 TB/s, where a large read reaches 6.1; the joining launch takes 4 more), a chain of
// latencies where they are few (16 ragged sessions of 512 to 8192 keys, 7B, 34 MB: 16 us and 4; of
// a workgroup's 11: 1.3 until it knows its part, 1.7 until the queries are in terms, 4.7 for 2 or 3
// tiles a wave, 1.9 for the end, the rest and the launch's other 5 not taken apart).  Pages that no cache holds cost
// little: the same call over 28 layers of a pool of 1 GB in turn 18.2 us instead of 17.6.  Many columns: vector and matrix instructions, which a SIMD
// hardly overlaps (8 x 512 rows behind up to 4096 keys, 7B, 122 GFLOP of scores and outputs: 241
// us, 506 TFLOP/s; per tile and wave 216 vector and 52 matrix instructions and 110 others take 960 ns
// of a SIMD, where the vector and matrix ones alone, on registers, take 678).  Left out one by
// one, the barrier is worth 4% of the time, three quarters of the LDS reads 2%, of K's loads nothing,
// 16 of the 52 products or the conversion of V 9% each.  Tiles in bf16: one in each session costs 2% of the many
// columns and nothing of the decodes; all of them (a token 2^-12 as large as the others in each) 8 x 512
// rows 366 us instead of 238, 8 x 32768 keys 68 instead of 62, 16 ragged sessions 19.3 instead of 17.5, 1 to 8 rows
// of 16 sessions 40.2 instead of 31.9.  Three waves a SIMD, and the next tile's
// scores under the softmax, are slower for want of registers.
#include <hip/hip_runtime.h>
#include <cstdint>
#include <type_traits>

namespace nova {
namespace {
// Batch of 8 x 512 rows (7B), 12 prompts of up to 300 rows (1.5B), 16 sessions of 1 to 8 rows (7B), us.
// kMinPiece 1: 245, 46.9, 34.3; 2: 243, 39.9, 32.6; 3: 242, 36.8, 32.5; 6: 240, 35.9, 35.8.
constexpr int kMinPiece = 3;
// A group's start (table, pages, queries in terms) and end against its tiles of 2 us.  0: 263, 45.2, 34.4;
// 1: 258, 41.2, 33.3; 2: 252, 38.9, 33.9; 4: 249, 36.6, 32.7.
constexpr int kGroupTiles = 4;
}  // namespace
}  // namespace nova

#include "attn_ragged.h"
#include "check.h"
#include "kv_q4.h"
#include "model.h"
#include "nova_kernel.h"

namespace nova {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u6 __attribute__((ext_vector_type(6)));
typedef int i8v __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f32v __attribute__((ext_vector_type(32)));

constexpr float kLow = 2.f, kSet = 10.f, kHigh = 15.9f;   // log2 of a tile's largest weight in fp16 terms: at least, where it is put, at most
constexpr float kLazy = 8.f;                   // and at most in bf16 terms: 2^21 products of the largest values stay inside fp32
constexpr float kDrop = 80.f;
constexpr int kCus = kAimWgs / 2;
constexpr int kSpread = 8;                     // powers of two of a tile in fp16: this many in a row
// Exponent bytes whose values (1/2 to 6 times the power) are normal numbers of fp16.  Subnormal ones would be
// exact too, but the matrix unit adds products up at the place of their operands' exponents, which it takes as
// fp16's least there: weights lose a bit for each power below (values of 2^-24, one after another: the result was
// off by 2^-12 of itself; of 2^-14 by 2^-20, as at any larger power).
constexpr int kLeastHalf = 127 - 13, kMostHalf = 127 + 13;
constexpr int kTerms = 5;                      // of the query
constexpr int kLeastExp = -100;                // of a query block: its last term's power is a normal number

// ---- operands ----

// A column's query, 1/sqrt(HD) and log2 e included, in kTerms terms of 6 bits.  Lane (g, c)
// holds dims 32 g .. + 31 of column c, the block that one power of two serves.
struct QTerms {
    u6 d[kTerms];
    int ex[kTerms];            // exponent bytes of the terms, each 5 less than the one before
};

__device__ __forceinline__ void q_terms(const f4 (&x)[8], QTerms& out) {
    uint32_t top = 0;
    f16v even, odd;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float y = x[j][e] * (kScale * kLog2e);
            top = max(top, __float_as_uint(y) & 0x7fffffffu);
            if (e & 1) odd[2 * j + e / 2] = y;
            else even[2 * j + e / 2] = y;
        }
    const bool finite = top < 0x7f800000u;
    const int ex = max((int)(top >> 23) - 127, kLeastExp);   // largest < 2^(ex + 1)
#pragma unroll
    for (int t = 0; t < kTerms; ++t) out.ex[t] = finite ? ex + 127 - 5 * t : kQ4Nan;
#pragma unroll
    for (int t = 0; t < kTerms; ++t) {
        const float unit = __uint_as_float((uint32_t)(ex + 127 - 5 * t) << 23);
        // elements 2 i, 2 i + 1 of the result: even[i], odd[i]
        u6 w = __builtin_amdgcn_cvt_scalef32_2xpk16_fp6_f32(even, odd, unit);
        // the conversion writes its result while it still reads: its operands are kept
        // past it, so that the two never share registers
        asm volatile("" : "+v"(w) : "v"(even), "v"(odd), "v"(unit));
        out.d[t] = w;
        if (t + 1 < kTerms) {
            f32v back = __builtin_amdgcn_cvt_scalef32_pk32_f32_fp6(w, unit);
            asm volatile("" : "+v"(back) : "v"(w), "v"(unit));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                even[i] -= back[2 * i];
                odd[i] -= back[2 * i + 1];
            }
        }
    }
}

// The query rows of a block's column, lane (g, c) its dims 32 g .. + 31.
__device__ __forceinline__ void load_q(const AttnArgs& a, const Session& s, int kvh, int col, f4 (&x)[8], int& seen) {
    const bool real = col < s.rows * G;
    const int r = real ? col / G : 0, hh = real ? col - r * G : 0;
    const float* src = a.q + ((int64_t)(s.row0 + r) * NH + kvh * G + hh) * HD + 32 * ((threadIdx.x & 63) >> 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = *reinterpret_cast<const f4*>(src + 4 * j);
        if (!real) x[j] = f4{0.f, 0.f, 0.f, 0.f};
    }
    seen = real ? min(s.past + r + 1, s.keys) : 0;
}

// fp4 rows of K (A) by 6-bit rows of the query (B), 128 dims; byte kByte of ke: the lane's K exponent
template <int kByte>
__device__ __forceinline__ f4 product(i4 k, u6 q, f4 z, int ke, int qe) {
    const i8v a = i8v{k[0], k[1], k[2], k[3], 0, 0, 0, 0};
    const i8v b = i8v{(int)q[0], (int)q[1], (int)q[2], (int)q[3], (int)q[4], (int)q[5], 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, z, 4, 2, kByte, ke, 0, qe);
}

// byte kByte of w as a power of two, for instructions that look at the exponent bits only
template <int kByte>
__device__ __forceinline__ float exponent_of(uint32_t w) {
    return __uint_as_float(kByte == 3 ? w >> 1 : w << (23 - 8 * kByte));
}

template <bool kHalf, int kByte>
__device__ __forceinline__ uint32_t pair_of(uint32_t w, uint32_t e) {
    if constexpr (kHalf) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, exponent_of<kByte>(e), kByte));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, exponent_of<kByte>(e), kByte));
}

// V of 4 tokens and two dims (32 b + r, 32 b + 16 + r) in fp16 or bf16: a byte of `w` per token,
// low half the lower dim; e: exponents, a byte per token.  Both dims of a token in a word.
template <bool kHalf>
__device__ __forceinline__ void pairs_of(uint32_t w, uint32_t e, uint32_t (&p)[4]) {
    each<4>([&](auto t) { p[t] = pair_of<kHalf, t>(w, e); });
}
// 8 tokens of either dim
__device__ __forceinline__ void by_dim(const uint32_t (&p)[4], const uint32_t (&q)[4], u4& lower, u4& upper) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        lower[i] = __builtin_amdgcn_perm(p[2 * i + 1], p[2 * i], 0x05040100u);
        upper[i] = __builtin_amdgcn_perm(p[2 * i + 1], p[2 * i], 0x07060302u);
        lower[2 + i] = __builtin_amdgcn_perm(q[2 * i + 1], q[2 * i], 0x05040100u);
        upper[2 + i] = __builtin_amdgcn_perm(q[2 * i + 1], q[2 * i], 0x07060302u);
    }
}
template <bool kHalf>
__device__ __forceinline__ void values_of(uint32_t w0, uint32_t w1, uint32_t e0, uint32_t e1, u4& lower, u4& upper) {
    uint32_t p[4], q[4];
    pairs_of<kHalf>(w0, e0, p);
    pairs_of<kHalf>(w1, e1, q);
    by_dim(p, q, lower, upper);
}

// 8 tokens' values (A) by their weights (B), added to z
template <bool kHalf>
__device__ __forceinline__ f4 add_up(u4 v, u4 w, f4 z) {
    if constexpr (kHalf) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, v), __builtin_bit_cast(h8, w), z, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, v), __builtin_bit_cast(b8, w), z, 0, 0, 0);
}

// Terms of the weights: two of fp16, cut off (the second ends at 2^-24), or the three of
// bf16 that are the weight's bits from the top, 8 at a time.
template <bool kHalf>
constexpr int kParts = kHalf ? 2 : 3;
template <bool kHalf>
__device__ __forceinline__ void split(const float (&e)[8], u4 (&w)[kParts<kHalf>]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        float a = e[j], b = e[j + 1];
        if constexpr (kHalf) {
            const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
            // what is left, a - h[0] and b - h[1], exact: one operation on the half as it is
            // (the compiler converts it first)
            float ra, rb;
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(h), "v"(a));
            asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(h), "v"(b));
            w[0][j / 2] = h;
            w[1][j / 2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(ra, rb));
        } else {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                w[k][j / 2] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
                if (k < 2) {
                    a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
                    b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
                }
            }
        }
    }
}

// The tokens of four exponent bytes that are NaN, as four bits; their bytes become 0 (the
// value counts through its weight instead).
__device__ __forceinline__ uint32_t take_nan(uint32_t& w) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if ((w >> (8 * k) & 255u) == (uint32_t)kQ4Nan) {
            m |= 1u << k;
            w &= ~(255u << (8 * k));
        }
    return m;
}

// The window of exponent bytes that tiles in fp16 lie in: `base` to base + kSpread - 1.
struct Window {
    uint32_t add, want, fill;  // per byte: what is added to a byte of the window gives `want` in its upper five bits
    bool closed;               // a value past fp16 is in the sums: no more fp16, so that the reference's drop keeps them finite
    __device__ __forceinline__ void at(int base) {
        const uint32_t b = (uint32_t)__builtin_amdgcn_readfirstlane(base), up = -b & (kSpread - 1);
        add = up * 0x01010101u;
        want = (b + up) * 0x01010101u;
        fill = b * 0x01010101u;
    }
    __device__ __forceinline__ void clear() {
        closed = false;
        at(127 - kSpread / 2);
    }
    // 0 where the four bytes lie in it (a byte that carries into the next one is itself outside)
    __device__ __forceinline__ uint32_t outside(uint32_t w) const { return ((w + add) ^ want) & 0xf8f8f8f8u; }
    // Moved to what a tile has, smallest and largest byte: true if that fits a window
    __device__ __forceinline__ bool move(int least, int most) {
        least = __builtin_amdgcn_readfirstlane(least);       // (the same in all lanes)
        most = __builtin_amdgcn_readfirstlane(most);
        if (most > kMostHalf) closed = true;
        const bool fits = !closed && most - least < kSpread && least >= kLeastHalf;
        if (fits) at(min(max((least + most + 1 - kSpread) / 2, kLeastHalf), kMostHalf + 1 - kSpread));
        return fits;
    }
};
static_assert(kSpread == 8, "upper five bits");

// smallest and largest of a lane's bytes that `keep` keeps, into the running ones
__device__ __forceinline__ void byte_range(uint32_t w, uint32_t keep, int& least, int& most) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        least = min(least, (int)((w | ~keep) >> (8 * k) & 255u));
        most = max(most, (int)((w & keep) >> (8 * k) & 255u));
    }
}
// of the exponents of four tokens, those of the first `rest`: slots behind the last key may hold anything
__device__ __forceinline__ uint32_t tokens_of(int rest) { return rest >= 4 ? ~0u : rest <= 0 ? 0u : (1u << (8 * rest)) - 1u; }
__device__ __forceinline__ void wave_range(int& least, int& most) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        least = min(least, __shfl_xor(least, o, 64));
        most = max(most, __shfl_xor(most, o, 64));
    }
}

// A block's state over the keys seen so far: lane (g, c) holds the reference, its share of
// the sum and dims 16 d + 4 g .. + 3 of column c.  `low` and `high`: between these a tile's
// largest score, less the reference, leaves it where it is (a column's first one moves it); top:
// the largest score that it was moved for.
struct State {
    float m, l, low, high, top;
    f4 acc[DB];
    __device__ __forceinline__ void clear() {
        m = l = 0.f;
        low = top = high = -INFINITY;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = f4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ bool unset() const { return high == -INFINITY; }
    __device__ __forceinline__ float reference() const { return unset() ? kUnset : m; }
    // the reference by `by` up or down for columns that move; z: scores less it
    __device__ __forceinline__ void move(bool moves, float col_top, float by, f4 (&z)[4]) {
        const float corr = !moves ? 1.f : unset() ? 0.f : __builtin_amdgcn_exp2f(-by);
        if (moves) {
            top = fmaxf(top, m + col_top);
            m += by;
            high = kHigh;
            low = m > top - kDrop ? kLow : -INFINITY;
        }
        l *= corr;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] *= corr;
#pragma unroll
        for (int u = 0; u < 4; ++u) z[u] -= moves ? by : 0.f;
    }
};

// Scores of one tile and block less the reference m.  k[u]: K operand of key block u (row
// 4p + i: token 4u + i of page p), ke: the exponents of its four key blocks.  Token j of the lane's
// page in z[j / 4][j % 4].  The sums begin at -m and take the query's largest term first:
// where the score is near m, and its weight counts, the others are added to a small number.
__device__ __forceinline__ void scores(const i4 (&k)[4], const QTerms& q, int ke, float m, f4 (&z)[4]) {
    const f4 from = f4{-m, -m, -m, -m};
#pragma unroll
    for (int t = 0; t < kTerms; ++t) {
        z[0] = product<0>(k[0], q.d[t], t ? z[0] : from, ke, q.ex[t]);
        z[1] = product<1>(k[1], q.d[t], t ? z[1] : from, ke, q.ex[t]);
        z[2] = product<2>(k[2], q.d[t], t ? z[2] : from, ke, q.ex[t]);
        z[3] = product<3>(k[3], q.d[t], t ? z[3] : from, ke, q.ex[t]);
    }
}

// scores of keys that the column does not see; key0: first key of the lane's page
__device__ __forceinline__ void hide(f4 (&z)[4], int key0, int seen) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
        if (key0 + j >= seen) z[j / 4][j % 4] = -INFINITY;
}

// The reference follows a tile's scores.
template <bool kHalf>
__device__ __forceinline__ void follow(f4 (&z)[4], State& st) {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; ++j) top = fmaxf(top, z[j / 4][j % 4]);
    if constexpr (kHalf) {
        // some lane above, or a column none of whose lanes is high enough
        uint64_t fine = __builtin_amdgcn_ballot_w64(top >= st.low);
        fine |= fine >> 32;
        fine |= fine >> 16;
        if (__builtin_amdgcn_ballot_w64(top > st.high) | (~fine & 0xffffu)) {
            const float col_top = rows_max(top);
            // (down no further than kDrop below the top)
            const float by = fmaxf(col_top - kSet, fminf(fmaxf(st.top - st.m, col_top) - kDrop, 0.f));
            st.move(col_top > -INFINITY && (col_top > st.high || (col_top < st.low && by < 0.f)), col_top, by, z);
        }
    } else {
        if (__builtin_amdgcn_ballot_w64(top > st.high - (kHigh - kLazy))) {
            const float col_top = rows_max(top);
            st.move(col_top > st.high - (kHigh - kLazy), col_top, col_top, z);
        }
    }
}

// Weights; nan: tokens of the lane's page whose value is NaN (bit per token; bf16 tiles only).
template <bool kHalf>
__device__ __forceinline__ void weights(const f4 (&z)[4], uint32_t nan, float (&e)[2][8]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) e[j / 8][j % 8] = __builtin_amdgcn_exp2f(z[j / 4][j % 4]);
    if (!kHalf && __builtin_amdgcn_ballot_w64(nan != 0))     // a seen value that is NaN makes the row NaN
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if ((nan >> j & 1) && z[j / 4][j % 4] > -INFINITY) e[j / 8][j % 8] = __builtin_nanf("");
}

__device__ __forceinline__ float sum_of(const float (&e)[2][8]) {
    float sum[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = (e[0][j] + e[0][4 + j]) + (e[1][j] + e[1][4 + j]);
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

__device__ __forceinline__ Session uniform(const Session& s) {
    return Session{__builtin_amdgcn_readfirstlane(s.keys), __builtin_amdgcn_readfirstlane(s.past),
                   __builtin_amdgcn_readfirstlane(s.rows), __builtin_amdgcn_readfirstlane(s.row0)};
}

// ---- few columns ----
//
// 16 columns (query rows x heads of a kv head) of a session's `blocks` times 16: the workgroup's
// waves share them and each takes its own keys, 64 at a time.  The operands come straight
// from the pages; the next tile's loads go out behind the products that have read their
// registers.  Blocks of 16 are workgroups of their own, which find each other's K and V in the
// caches: two blocks in one take the registers of one wave a SIMD and, at 4 rows of 7B, 18.5 us
// instead of 15.6 behind 8 x 2000 keys, 34.8 instead of 23.6 behind 4 x 16000.  kOnce: non-temporal
// loads, for pools that no cache holds until the next step; solo: no cuts (see launch()).
template <bool kCausal, bool kOnce, int kWaves>
__global__ void __launch_bounds__(64 * kWaves, 2) q4_few_kernel(AttnArgs a, int blocks, bool solo) {
    __shared__ __attribute__((aligned(16))) float s_acc[kWaves][16][kAccRow];
    __shared__ float s_m[kWaves][16], s_l[kWaves][16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int kvh = blockIdx.x % NKV, unit = blockIdx.x / NKV;
    const int slot = unit / blocks, col0 = 16 * (unit - slot * blocks);      // the first of the workgroup's columns
    Part p;
    const bool whole = solo && a.table_stride <= 64;         // a lane per page of the table:
    int row = 0;                                             // its row, requested beside the length
    if (solo) {                                              // a slot per session
        if (whole) row = a.tables[slot * a.table_stride + min(lane, (int)a.table_stride - 1)];
        p = Part{slot, 0, 1, uniform(session_of<kCausal>(a, slot))};
        if (p.s.rows * G <= col0) return;
    } else {
        p = find_part<kCausal>(a, slot);
        if (p.sess < 0 || p.s.rows * G <= col0) return;
    }
    if (!solo && kvh == 0 && col0 == 0 && p.index == 0 && tid == 0) a.info[p.sess] = i4{slot, p.parts, p.s.rows, p.s.row0};
    const int n_cols = min(p.s.rows * G - col0, 16);
    // the part's tiles, and this wave's of them
    const int tiles = (p.s.keys + TILE - 1) / TILE;
    const int t_lo = (int)((int64_t)tiles * p.index / p.parts), t_hi = (int)((int64_t)tiles * (p.index + 1) / p.parts);
    const int t0 = t_lo + (t_hi - t_lo) * wave / kWaves, t1 = t_lo + (t_hi - t_lo) * (wave + 1) / kWaves;
    const int clear_keys = min(p.s.past + col0 / G + 1, p.s.keys);           // keys below: seen by all its columns

    // lane (g, c) reads K rows and exponents of page c >> 2, V columns and exponents of page g
    Pages pages(a, p.sess, p.s.keys);
    if (whole) {
        pages.win = 0;
        pages.held = row;
    }
    const uint8_t *k_at = nullptr, *v_at = nullptr;
    i4 kr[4], vr[4];
    int ke = 0, ve = 0;
    auto load_k = [&](int t) {
        const int pg = t * kTilePages;
        pages.reach(pg);
        const uint8_t* head = a.pool + kvh * kQ4Rec;
        k_at = head + pages[pg + (c >> 2)] * kQ4Page + (c & 3) * 64 + g * 16;
        v_at = head + pages[pg + g] * kQ4Page;
#pragma unroll
        for (int u = 0; u < 4; ++u) kr[u] = page_load<kOnce>(k_at + 256 * u);
        ke = *reinterpret_cast<const int*>(k_at - (c & 3) * 48 - g * 12 + kQ4KeOff);     // (c & 3) * 16 + g * 4 of the page's
        ve = *reinterpret_cast<const int*>(v_at + kQ4VeOff + 4 * c);
    };
    auto load_v = [&] {
#pragma unroll
        for (int b = 0; b < 4; ++b) vr[b] = page_load<kOnce>(v_at + kQ4VOff + 256 * b + 16 * c);
    };
    QTerms q;
    State st;
    int seen;                  // keys that the column sees
    Window win;
    win.clear();
    st.clear();
    if (t0 < t1) {             // the queries first: they have come when the first pages are on their way
        f4 x[8];
        load_q(a, p.s, kvh, col0 + c, x, seen);
        load_k(t0);
        load_v();
        q_terms(x, q);
    }
    auto step = [&](auto mask_tag, int t) {
        constexpr bool kMask = decltype(mask_tag)::value;
        const int key0 = t * TILE + 16 * g;
        uint32_t ex = (uint32_t)ve, keep = ~0u;              // the lane's: tokens 4 (c & 3) .. of block c >> 2
        if (kMask) {
            keep = tokens_of(p.s.keys - key0 - 4 * (c & 3));
            ex = (ex & keep) | (win.fill & ~keep);
        }
        auto rest = [&](auto half_tag, uint32_t nan) {
            constexpr bool kHalf = decltype(half_tag)::value;
            constexpr int kN = kParts<kHalf>;
            u4 w[2][kN];
            f4 z[4];
            float e[2][8];
            scores(kr, q, ke, st.m, z);
            if (kMask) hide(z, key0, seen);
            follow<kHalf>(z, st);
            weights<kHalf>(z, nan, e);
            st.l += sum_of(e);
            split<kHalf>(e[0], w[0]);
            split<kHalf>(e[1], w[1]);
            const bool more = t + 1 < t1;
            if (more) load_k(t + 1);
            each<4>([&](auto b) {
                constexpr int kB = b;
                uint32_t e[4];
                each<4>([&](auto i) { e[i] = __float_as_uint(row_lane<4 * kB + i>(__uint_as_float(ex))); });
                each<2>([&](auto h) {
                    u4 lower, upper;
                    values_of<kHalf>((uint32_t)vr[b][2 * h], (uint32_t)vr[b][2 * h + 1], e[2 * h], e[2 * h + 1], lower, upper);
#pragma unroll
                    for (int k = kN - 1; k >= 0; --k) {
                        st.acc[2 * b] = add_up<kHalf>(lower, w[h][k], st.acc[2 * b]);
                        st.acc[2 * b + 1] = add_up<kHalf>(upper, w[h][k], st.acc[2 * b + 1]);
                    }
                });
            });
            if (more) load_v();
        };
        bool half = !win.closed && __builtin_amdgcn_ballot_w64(win.outside(ex) != 0) == 0;
        uint32_t nan = 0;
        if (!half) {                                         // rare: another window, or none
            nan = take_nan(ex) << (4 * (c & 3));
            int least = 255, most = 0;
            byte_range(ex, keep, least, most);
            wave_range(least, most);
            half = win.move(least, most);                    // (not with NaN in it, whose bytes are 0 now)
            if (kMask) ex = (ex & keep) | (win.fill & ~keep);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) nan |= (uint32_t)__shfl_xor((int)nan, o, 64);
        }
        if (half) rest(std::true_type{}, 0u);
        else rest(std::false_type{}, nan);
    };
    const int t_clear = max(min(t1, clear_keys / TILE), t0);
    for (int t = t0; t < t_clear; ++t) step(std::false_type{}, t);
    for (int t = t_clear; t < t1; ++t) step(std::true_type{}, t);

    // the waves' states joined in LDS; a lone part writes the output
    const float sum_l = rows_sum(st.l);
    if (g == 0) {
        s_m[wave][c] = st.reference();
        s_l[wave][c] = sum_l;
    }
    if (c < n_cols)
#pragma unroll
        for (int d = 0; d < DB; ++d) *reinterpret_cast<f4*>(&s_acc[wave][c][16 * d + 4 * g]) = st.acc[d];
    __syncthreads();
    for (int e = tid; e < n_cols * (HD / 4); e += 64 * kWaves) {
        const int cc = e / (HD / 4), d4 = e % (HD / 4), col = col0 + cc;
        float m = s_m[0][cc];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_m[w][cc]);
        f4 sum = f4{0.f, 0.f, 0.f, 0.f};
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const Factor f(s_m[w][cc] - m);
            sum += f * *reinterpret_cast<const f4*>(&s_acc[w][cc][4 * d4]);
            l += f * s_l[w][cc];
        }
        if (p.parts == 1) {
            const int r = col / G, hh = col - r * G;
            const float n = p.s.keys > 0 ? 1.0f / l : 0.f;
            *reinterpret_cast<f4*>(a.o + ((int64_t)(p.s.row0 + r) * NH + kvh * G + hh) * HD + 4 * d4) = sum * n;
        } else {
            const int64_t at = ((int64_t)kvh * a.slots + slot) * (16 * blocks) + col;
            *reinterpret_cast<f4*>(a.acc + at * HD + 4 * d4) = sum;
            if (d4 == 0) a.ml[at] = f2{m, l};
        }
    }
}

// ---- many columns ----

// Each wave has its own 16 columns of a group, and all go over the same keys.  A wave takes K
// from the pages to its registers (the four of a workgroup find it in the caches), so its scores and
// weights wait for nobody; V's conversion is done once for 64 columns: wave w turns page w of a
// tile into fp16 (or bf16) in operand order in LDS, two tiles of it.  A tile's loads go out
// while the one before it is worked on; one barrier per tile, between the weights and the products
// that they go into.  All waves see the exponents of the whole tile, so they agree on
// its type without a word.
__global__ void __launch_bounds__(THREADS, 2) q4_many_kernel(AttnArgs a) {
    constexpr int COLS = kManyCols;
    constexpr int kOut = 16 * kAccRow * 4;                   // a block's results, per wave
    constexpr int kVTile = 2 * DB * 1024;
    static_assert(kTilePages == WAVES, "a page per wave");
    constexpr int kMem = WAVES * kOut > 2 * kVTile ? WAVES * kOut : 2 * kVTile;      // the results overwrite the tiles
    __shared__ __attribute__((aligned(16))) unsigned char s_mem[kMem];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x, w = blockIdx.y;

    Place at, to;
    find_stretch(a, w, at, to);
    i4 piece[2] = {i4{-1, 0, 0, 0}, i4{-1, 0, 0, 0}};        // the group begun before this stretch; the one it leaves open
    Window win;
    win.clear();
    for (;;) {
        if (at.sess >= a.n_sess || at.sess > to.sess ||
            (at.sess == to.sess && (at.group > to.group || (at.group == to.group && at.tile >= to.tile))))
            break;
        const Session s = uniform(session_of<true>(a, at.sess));
        if (at.group >= n_groups(s)) {
            at = Place{at.sess + 1, 0, 0};
            continue;
        }
        // (a lane number that is new for each group: what is made of it is made again, and not kept
        // in registers that the tiles need, or behind them in memory)
        int lane = tid & 63;
        asm volatile("" : "+v"(lane));
        const int g = lane >> 4, c = lane & 15;
        const int sess = at.sess, group = at.group;
        const int tiles = __builtin_amdgcn_readfirstlane(group_tiles(s, group));
        const int t_lo = __builtin_amdgcn_readfirstlane(at.tile);
        const int t_hi = __builtin_amdgcn_readfirstlane(sess == to.sess && group == to.group ? to.tile : tiles);
        at = Place{sess, group + 1, 0};
        if (t_lo >= t_hi) continue;

        const int n_cols = s.rows * G, col0 = group * COLS + wave * 16;
        const int wave_keys = col0 < n_cols ? min(s.past + min(col0 + 15, n_cols - 1) / G + 1, s.keys) : 0;
        const int t1 = __builtin_amdgcn_readfirstlane(min(t_hi, (wave_keys + TILE - 1) / TILE));   // this wave's last tile
        const int t_clear = __builtin_amdgcn_readfirstlane(min(s.past + col0 / G + 1, s.keys) / TILE);   // tiles below: seen by all its columns

        // ---- a tile's way to the wave ----
        Pages pages(a, sess, s.keys);
        const uint8_t* const head = a.pool + kvh * kQ4Rec;
        i4 kr[4], vr, ve;                                    // K of the tile; V of page `wave` and its exponents of block g
        int ke = 0;
        uint32_t vx = 0;                                     // V's exponents of the tile: page c >> 2, block g, tokens 4 (c & 3) ..
        struct Where {
            int lane, wave;                                  // pages of the pool: c >> 2 of a tile, and `wave`
        };
        auto where = [&](int t) {
            const int pg = t * kTilePages;
            pages.reach(pg);
            const int own = __builtin_amdgcn_readlane(pages.held, min(pg + wave, pages.last) - pages.win);
            return Where{pages[pg + (c >> 2)], (unsigned)own < (unsigned)a.nb ? own : 0};
        };
        auto load_v = [&](const Where& at) {
            const uint8_t* rec = head + at.wave * kQ4Page;
            vr = *reinterpret_cast<const i4*>(rec + kQ4VOff + 16 * lane);
            ve = *reinterpret_cast<const i4*>(rec + kQ4VeOff + 16 * g);
            vx = *reinterpret_cast<const uint32_t*>(head + at.lane * kQ4Page + kQ4VeOff + g * 16 + (c & 3) * 4);
        };
        auto load_k = [&](const Where& at) {
            const uint8_t* rec = head + at.lane * kQ4Page;
            const uint8_t* k_at = rec + (c & 3) * 64 + g * 16;
#pragma unroll
            for (int u = 0; u < 4; ++u) kr[u] = *reinterpret_cast<const i4*>(k_at + 256 * u);
            ke = *reinterpret_cast<const int*>(rec + kQ4KeOff + (c & 3) * 16 + g * 4);
        };
        // the exponents of tokens from..from + 3 with those of slots behind the last key, which
        // may hold anything, replaced
        auto cut = [&](uint32_t x, int from) {
            const uint32_t keep = tokens_of(s.keys - from);
            return (x & keep) | (win.fill & ~keep);
        };
        // V of a tile in operand order, lane (g, c) dims 32 g + c and 32 g + 16 + c of page `wave`; to LDS
        auto turn = [&](auto half_tag, u4 (&v)[2][2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                values_of<decltype(half_tag)::value>((uint32_t)vr[2 * h], (uint32_t)vr[2 * h + 1], (uint32_t)ve[2 * h],
                                                     (uint32_t)ve[2 * h + 1], v[0][h], v[1][h]);
        };
        auto write_v = [&](const u4 (&v)[2][2], int t) {
            unsigned char* dst = s_mem + (t & 1) * kVTile + g * 4096 + (16 * wave + c) * 16;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int h = 0; h < 2; ++h) *reinterpret_cast<u4*>(dst + x * 2048 + h * 1024) = v[x][h];
        };
        uint32_t nan = 0;                                    // tokens of page g whose value is NaN
        // the same for any tile; true: in fp16
        auto put = [&](int t) {
            const int from = t * TILE + 16 * (c >> 2) + 4 * (c & 3);
            uint32_t x = cut(vx, from);
            auto cut_own = [&] {
#pragma unroll
                for (int i = 0; i < 4; ++i) ve[i] = (int)cut((uint32_t)ve[i], t * TILE + 16 * wave + 4 * i);
            };
            cut_own();
            bool half = !win.closed && __builtin_amdgcn_ballot_w64(win.outside(x) != 0) == 0;
            nan = 0;
            if (!half) {                                     // another window, or none
                const uint32_t m = take_nan(x) << (4 * (c & 3));
                int least = 255, most = 0;
                byte_range(x, tokens_of(s.keys - from), least, most);
                wave_range(least, most);
                half = win.move(least, most);                // (not with NaN in it, whose bytes are 0 now)
                cut_own();
                if (__builtin_amdgcn_ballot_w64(m != 0)) {
                    nan = m;
                    nan |= (uint32_t)__shfl_xor((int)nan, 1, 64);
                    nan |= (uint32_t)__shfl_xor((int)nan, 2, 64);
                    nan |= (uint32_t)__shfl_xor((int)nan, 16, 64);
                    nan |= (uint32_t)__shfl_xor((int)nan, 32, 64);
                    nan = (uint32_t)__shfl((int)nan, 4 * g, 64);             // page c >> 2 -> page g
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t y = (uint32_t)ve[i];
                        (void)take_nan(y);
                        ve[i] = (int)y;
                    }
                }
            }
            u4 v[2][2];
            if (half) turn(std::true_type{}, v);
            else turn(std::false_type{}, v);
            write_v(v, t);
            return half;
        };
        // the wave's LDS accesses are done; loads in flight stay there
        auto barrier = [&] {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        QTerms q;
        int seen;
        State st;
        const Where start = where(t_lo);
        {
            f4 x[8];
            load_q(a, s, kvh, col0 + c, x, seen);
            load_v(start);
            load_k(start);
            q_terms(x, q);
            st.clear();
            win.closed = false;                              // (the window stays: it says nothing about the sums)
        }
        // One tile: its scores and weights, then the barrier that V waits for, then its
        // products.  True: V of the next tile is in LDS as well, in fp16 (what almost all are).
        // (Behind the last tile the same once more: no branch, so that the registers stay where
        // they are.)
        auto tile = [&](auto half_tag, int t) {
            constexpr bool kHalf = decltype(half_tag)::value;
            constexpr int kN = kParts<kHalf>;
            const Where next = where(min(t + 1, t_hi - 1));
            load_v(next);
            f4 z[4];
            float e[2][8];
            scores(kr, q, ke, st.m, z);
            __builtin_amdgcn_sched_barrier(0);               // K's registers are free now
            // vector work goes first: the other workgroup's products run beside it (batch 240 us;
            // 248 without, 244 the other way round)
            __builtin_amdgcn_s_setprio(1);
            load_k(next);
            if (t >= t_clear) hide(z, t * TILE + 16 * g, seen);
            follow<kHalf>(z, st);
            weights<kHalf>(z, nan, e);
            st.l += sum_of(e);
            __builtin_amdgcn_s_setprio(0);
            barrier();
            const unsigned char* v_at = s_mem + (t & 1) * kVTile + 16 * lane;
            u4 p[2][kN];
            split<kHalf>(e[0], p[0]);
            split<kHalf>(e[1], p[1]);
#pragma unroll
            for (int d = 0; d < DB; d += 2) {                // two 16-dim blocks, two halves of their tokens
                u4 v[2][2];
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h) v[x][h] = *reinterpret_cast<const u4*>(v_at + 1024 * (2 * (d + x) + h));
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = kN - 1; k >= 0; --k)
#pragma unroll
                        for (int x = 0; x < 2; ++x) st.acc[d + x] = add_up<kHalf>(v[x][h], p[h][k], st.acc[d + x]);
            }
            // (the last tile, whose page may end behind the last key, goes the other way)
            if (!kHalf || t + 1 >= t1 || (t + 2) * TILE > s.keys || __builtin_amdgcn_ballot_w64(win.outside(vx) != 0) != 0)
                return false;
            u4 w[2][2];
            turn(std::true_type{}, w);
            write_v(w, t + 1);
            return true;
        };
        // Every wave goes through all tiles of the stretch, for its page of them and the
        // barrier; its own columns need the first ones, up to t_clear without a mask.
        for (int t = t_lo; t < t_hi; ++t) {
            const bool half = put(t);
            if (t < t1 && half) {
                while (tile(std::true_type{}, t)) ++t;
            } else if (t < t1) {
                tile(std::false_type{}, t);
            } else {
                load_v(where(min(t + 1, t_hi - 1)));
                barrier();
            }
        }
        barrier();                                           // all waves are past their products

        // results through LDS (every wave is past its tiles), rows in address order:
        // the output, or a piece of a group that others have the rest of
        const bool whole = t_lo == 0 && t_hi == tiles;
        const int slot = 2 * w + (t_lo > 0 ? 0 : 1);
        if (!whole) piece[t_lo > 0 ? 0 : 1] = i4{sess, group, t_hi == tiles, min(n_cols - group * COLS, COLS)};
        unsigned char* mine = s_mem + wave * kOut;
        asm volatile("" : "+v"(lane));
        if (col0 < n_cols) {
            const float l = rows_sum(st.l), m = st.reference();
#pragma unroll
            for (int d = 0; d < DB; ++d) *reinterpret_cast<f4*>(mine + ((lane & 15) * kAccRow + 16 * d + 4 * (lane >> 4)) * 4) = st.acc[d];
            wave_lds_sync();
#pragma unroll
            for (int e = 0; e < 16 * (HD / 4) / 64; ++e) {
                const int cc = 2 * e + lane / 32, d4 = lane % 32, col = col0 + cc;
                const f4 sum = *reinterpret_cast<const f4*>(mine + (cc * kAccRow + 4 * d4) * 4);
                const float cl = __shfl(l, cc, 64), cm = __shfl(m, cc, 64);
                if (col >= n_cols) continue;
                if (whole) {
                    const int r = col / G, hh = col - r * G;
                    *reinterpret_cast<f4*>(a.o + ((int64_t)(s.row0 + r) * NH + kvh * G + hh) * HD + 4 * d4) = sum * (1.0f / cl);
                } else {
                    const int64_t to_at = ((int64_t)kvh * a.slots + slot) * COLS + wave * 16 + cc;
                    *reinterpret_cast<f4*>(a.acc + to_at * HD + 4 * d4) = sum;
                    if (d4 == 0) a.ml[to_at] = f2{cm, cl};
                }
            }
        }
        barrier();                                           // the next group's tiles come where the results were
    }
    if (kvh == 0 && tid < 2) a.info[2 * w + tid] = tid ? piece[1] : piece[0];
}

// ---- host side ----

template <bool kCausal>
void launch(AttnArgs a, void* workspace, hipStream_t s) {
    const Shape f = shape(a.n_sess, a.max_q);
    const Layout w = layout(f, a.n_sess);
    char* ws = static_cast<char*>(workspace);
    a.slots = f.slots;
    a.info = reinterpret_cast<i4*>(ws + w.info);
    a.ml = reinterpret_cast<f2*>(ws + w.ml);
    a.acc = reinterpret_cast<float*>(ws + w.acc);
    const unsigned join_wgs = (unsigned)std::min<int64_t>((int64_t)a.rows.n_rows * NH, kJoinWgs);
    // Up to 64 columns of short tables: a workgroup per session, kv head and 16 columns, nothing to find and
    // nothing to join.  The table's width counts, as the host knows no lengths: 8 sessions of 300 keys (7B) 6.9 us over a
    // table of up to 64 pages, 9.5 over a wider one.  Up to 64 pages; where the workgroups are 64 and more, up to 96, as parts of the sessions
    // would share CUs.  One launch against two (us, one after another in a graph), 1 / 8 / 32 sessions of 7B: of 300
    // keys 6.6, 6.8, 6.9 against 9.2, 9.3, 10.0; of 1024 8.9, 9.2, 9.5 against 9.4, 9.6, 12.6; of 1040 10.5, 10.8, 11.2
    // against 9.5, 9.8, 14.0; of 1536 11.4, 11.7, 12.4 against 9.5, 9.8, 14.7.
    // 33 to 64 columns against the form of many: 8 rows behind 1 / 16 / 64 x 500 keys 8.1, 8.8, 21.3 and 16.6, 20.6,
    // 28.8; 64 x 1400 40.4 and 39.7; without the limit, 16 x 3000 of 5 rows, in parts, 28.4 and 25.3.
    const int64_t cols = (int64_t)a.max_q * G;
    const int blocks = cols <= 64 ? (int)(cols + 15) / 16 : 1;
    const int64_t wgs = (int64_t)a.n_sess * NKV * blocks;
    const bool solo = cols <= 64 && a.table_stride <= (wgs >= kCus / 4 ? 96 : 64);
    if constexpr (kCausal) {
        if (f.many && !solo) {
            hipLaunchKernelGGL(q4_many_kernel, dim3(NKV, a.gw), dim3(THREADS), 0, s, a);
            NOVA_LAUNCHED();
            hipLaunchKernelGGL(many_join_kernel, dim3(join_wgs), dim3(THREADS), 0, s, a);
            NOVA_LAUNCHED();
            return;
        }
    }
    // With a CU for each of them, eight waves instead of four (7.1 and 9.6 us for 16 sessions of 300 and 1024 keys of
    // 7B with four, 6.8 and 9.2 with eight).
    const bool wide = solo && wgs <= kCus;
    a.gw /= blocks;
    const dim3 grid((unsigned)(solo ? wgs : (int64_t)NKV * f.slots * blocks));   // (past what a second dimension holds)
    // The pages of a pool larger than the 256 MB memory-side cache (all layers of it,
    // as a step walks through them) come from HBM.
    const bool once = (int64_t)Model::L * a.nb * kQ4Page > (int64_t)256 << 20;
    auto run = [&](auto once_tag) {
        constexpr bool kOnce = decltype(once_tag)::value;
        if (wide) hipLaunchKernelGGL((q4_few_kernel<kCausal, kOnce, 8>), grid, dim3(512), 0, s, a, blocks, solo);
        else hipLaunchKernelGGL((q4_few_kernel<kCausal, kOnce, WAVES>), grid, dim3(THREADS), 0, s, a, blocks, solo);
    };
    if (once) run(std::true_type{});
    else run(std::false_type{});
    NOVA_LAUNCHED();
    if (solo) return;
    hipLaunchKernelGGL(few_join_kernel, dim3(join_wgs), dim3(THREADS), 0, s, a, f.cols);
    NOVA_LAUNCHED();
}

}  // namespace
}  // namespace nova

using namespace nova;

extern "C" {

size_t attn_decode_q4_workspace_bytes(int n_sess) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535);
    return layout(shape(n_sess, 1), n_sess).total;
}

size_t attn_chunk_q4_workspace_bytes(int n_sess, int n_rows, int max_q) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && n_rows >= 0 && max_q >= 0 && max_q <= n_rows);
    return layout(shape(n_sess, max_q), n_sess).total;
}

void launch_attn_decode_q4_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                 const int32_t* n_keys, int n_sess, int layer, int nb, float* o, void* workspace,
                                 nova_stream_t s) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535);
    AttnArgs a = attn_args(kQ4Page, q, pool, tables, table_stride, n_keys, n_sess, layer, nb, o);
    NOVA_REQUIRE(workspace && aligned16(workspace));
    a.rows = RaggedRows{nullptr, 1, n_sess};
    a.max_q = 1;
    launch<false>(a, workspace, reinterpret_cast<hipStream_t>(s));
}

void launch_attn_chunk_q4_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                const int32_t* n_past, const int32_t* row_off, int n_sess, int n_rows, int max_q,
                                int layer, int nb, float* o, void* workspace, nova_stream_t s) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && n_rows >= 0 && n_rows <= (1 << 24));
    NOVA_REQUIRE(max_q >= 0 && max_q <= n_rows);
    NOVA_REQUIRE(row_off || n_rows % n_sess == 0);
    AttnArgs a = attn_args(kQ4Page, q, pool, tables, table_stride, n_past, n_sess, layer, nb, o);
    NOVA_REQUIRE(workspace && aligned16(workspace));
    if (n_rows == 0 || max_q == 0) return;
    a.rows = RaggedRows{row_off, n_rows / n_sess, n_rows};
    a.max_q = max_q;
    launch<true>(a, workspace, reinterpret_cast<hipStream_t>(s));
}

}  // extern "C"
