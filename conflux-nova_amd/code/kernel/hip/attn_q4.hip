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
// sums are fp32.  V becomes bf16 with its power of two, which is exact, and a weight is
// the exact sum of three bf16 terms (8 bits each), so the products lose nothing and their
// sums are fp32.
//
// One pass over the keys with a running reference and sum of the softmax.  The reference
// of the weights 2^(s - m) follows the largest score lazily: a weight may grow to
// 2^kLazy before the sums are rescaled, so that almost no tile does it.
#include <hip/hip_runtime.h>
#include <cstdint>
#include <type_traits>

#include "attn_ragged.h"
#include "check.h"
#include "kv_q4.h"
#include "model.h"
#include "nova_kernel.h"

namespace nova {
namespace {

typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u6 __attribute__((ext_vector_type(6)));
typedef int i8v __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f32v __attribute__((ext_vector_type(32)));

constexpr float kLazy = 8.f;                   // log2 of a weight that may be above 1 so far
constexpr int kTerms = 5;                      // of the query
constexpr int kLeastExp = -100;                // of a query block: its last term's power is a normal number

// ---- operands ----

// A column's query, 1/sqrt(HD) and log2 e included, in kTerms terms of 6 bits.  Lane (g, c)
// holds dims 32 g .. + 31 of column c, the block that one power of two serves.
struct QTerms {
    u6 d[kTerms];
    int ex;                    // exponent byte of the first term; each one after it 5 less
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
    out.ex = finite ? ex + 127 : kQ4Nan;
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
__device__ __forceinline__ void load_q(const AttnArgs& a, const Session& s, int kvh, int col, QTerms& out, int& seen) {
    const bool real = col < s.rows * G;
    const int r = real ? col / G : 0, hh = real ? col - r * G : 0;
    const float* src = a.q + ((int64_t)(s.row0 + r) * NH + kvh * G + hh) * HD + 32 * ((threadIdx.x & 63) >> 4);
    f4 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = *reinterpret_cast<const f4*>(src + 4 * j);
        if (!real) x[j] = f4{0.f, 0.f, 0.f, 0.f};
    }
    q_terms(x, out);
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

// V of 8 tokens and two dims (32 b + r, 32 b + 16 + r): a byte of `w0`, `w1` per token, low
// half the lower dim; e0, e1: exponents, a byte per token
__device__ __forceinline__ void values_bf16(uint32_t w0, uint32_t w1, uint32_t e0, uint32_t e1, b8& lower, b8& upper) {
    uint32_t p[8];
    each<4>([&](auto t) {
        constexpr int kByte = t;
        p[t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w0, exponent_of<kByte>(e0), kByte));
        p[4 + t] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w1, exponent_of<kByte>(e1), kByte));
    });
    u4 lo, hi;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo[i] = __builtin_amdgcn_perm(p[2 * i + 1], p[2 * i], 0x05040100u);
        hi[i] = __builtin_amdgcn_perm(p[2 * i + 1], p[2 * i], 0x07060302u);
    }
    lower = __builtin_bit_cast(b8, lo);
    upper = __builtin_bit_cast(b8, hi);
}

// weights as the exact sums of three bf16 terms: their bits from the top, 8 at a time
__device__ __forceinline__ void split_bf16(const float (&e)[8], b8 (&out)[3]) {
    u4 w[3];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        float a = e[j], b = e[j + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            w[k][j / 2] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
            if (k < 2) {
                a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
                b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) out[k] = __builtin_bit_cast(b8, w[k]);
}

// which of the four bytes are 255, as bits 0, 8, 16, 24 (exact: the lowest of them and
// everything below it; those above may be wrong only where one below is right, so this asks
// byte by byte)
__device__ __forceinline__ uint32_t bytes_255(uint32_t w) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) m |= ((w >> (8 * k)) & 255u) == 255u ? 1u << (8 * k) : 0u;
    return m;
}
// quick: none of the bytes is 255 if this is 0
__device__ __forceinline__ uint32_t maybe_255(uint32_t w) { return (~w - 0x01010101u) & w & 0x80808080u; }

// A block's state over the keys seen so far: lane (g, c) holds the reference, its share of
// the sum and dims 16 d + 4 g .. + 3 of column c.  A score above `limit` moves the
// reference (a column's first one always does).
struct State {
    float m, l, limit;
    f4 acc[DB];
    __device__ __forceinline__ void clear() {
        m = l = 0.f;
        limit = -INFINITY;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = f4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ float reference() const { return limit == -INFINITY ? kUnset : m; }
};

// Scores, weights and sum of one tile and block.  k_op(u): K operand of key block u (row
// 4p + i: token 4u + i of page p), ke: the exponents of its four key blocks; key0: first key
// of the lane's page; nan: tokens of it whose value is NaN (bit per token; 0 in almost all tiles).
template <bool kMask, class K>
__device__ __forceinline__ void weigh(K&& k_op, const QTerms& q, int ke, int key0, int seen, uint32_t nan, State& st,
                                      b8 (&p)[2][3]) {
    f4 z[4];
    const i4 k[4] = {k_op(0), k_op(1), k_op(2), k_op(3)};
#pragma unroll
    for (int u = 0; u < 4; ++u) z[u] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = kTerms - 1; t >= 0; --t) {                  // the small terms first
        const int qe = q.ex == kQ4Nan ? kQ4Nan : q.ex - 5 * t;
        z[0] = product<0>(k[0], q.d[t], z[0], ke, qe);
        z[1] = product<1>(k[1], q.d[t], z[1], ke, qe);
        z[2] = product<2>(k[2], q.d[t], z[2], ke, qe);
        z[3] = product<3>(k[3], q.d[t], z[3], ke, qe);
    }
    float x[16];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        x[j] = z[j / 4][j % 4];
        if (kMask && key0 + j >= seen) x[j] = -INFINITY;
        top = fmaxf(top, x[j]);
    }
    if (__builtin_amdgcn_ballot_w64(top > st.limit)) {       // rare
        const float col_top = rows_max(top);
        const bool moves = col_top > st.limit, first = st.limit == -INFINITY;
        const float to = moves ? col_top : st.m;
        const float corr = first ? 0.f : __builtin_amdgcn_exp2f(st.m - to);
        st.m = to;
        st.limit = moves ? to + kLazy : st.limit;
        st.l *= corr;
#pragma unroll
        for (int d = 0; d < DB; ++d) st.acc[d] *= corr;
    }
    float e[2][8];
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        e[j / 8][j % 8] = __builtin_amdgcn_exp2f(x[j] - st.m);
        sum[j / 4] += e[j / 8][j % 8];
    }
    if (__builtin_amdgcn_ballot_w64(nan != 0))               // rare: a seen value that is NaN makes the row NaN
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if ((nan >> j & 1) && key0 + j < seen) e[j / 8][j % 8] = __builtin_nanf("");
    st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    split_bf16(e[0], p[0]);
    split_bf16(e[1], p[1]);
}

// ---- few columns ----
//
// Up to 16 NB columns (query rows x heads of a kv head) of a session: the workgroup's waves
// share them and each takes its own keys, 64 at a time, so K and V are read once.  The
// operands come straight from the pages; the next tile's loads go out behind the products
// that have read their registers.  kOnce: non-temporal loads, for pools that no cache
// holds until the next step (see launch()).
template <int NB, bool kCausal, bool kOnce>
__global__ void __launch_bounds__(THREADS, NB == 1 ? 2 : 1) q4_few_kernel(AttnArgs a) {
    constexpr int COLS = 16 * NB;
    __shared__ __attribute__((aligned(16))) float s_acc[WAVES][16][kAccRow];
    __shared__ float s_m[WAVES][COLS], s_l[WAVES][COLS];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int kvh = blockIdx.x, slot = blockIdx.y;
    const Part p = find_part<kCausal>(a, slot);
    if (p.sess < 0) return;
    if (kvh == 0 && p.index == 0 && tid == 0) a.info[p.sess] = i4{slot, p.parts, p.s.rows, p.s.row0};
    const int n_cols = p.s.rows * G;
    // the part's tiles, and this wave's of them
    const int tiles = (p.s.keys + TILE - 1) / TILE;
    const int t_lo = (int)((int64_t)tiles * p.index / p.parts), t_hi = (int)((int64_t)tiles * (p.index + 1) / p.parts);
    const int t0 = t_lo + (t_hi - t_lo) * wave / WAVES, t1 = t_lo + (t_hi - t_lo) * (wave + 1) / WAVES;
    const int clear_keys = min(p.s.past + 1, p.s.keys);      // keys below: seen by all columns

    // lane (g, c) reads K rows and exponents of page c >> 2, V columns and exponents of page g
    Pages pages(a, p.sess, p.s.keys);
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
    if (t0 < t1) {
        load_k(t0);
        load_v();
    }
    QTerms q[NB];
    int seen[NB];              // keys that the column sees
    State st[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        load_q(a, p.s, kvh, 16 * b + c, q[b], seen[b]);
        st[b].clear();
    }
    auto step = [&](auto mask_tag, int t) {
        constexpr bool kMask = decltype(mask_tag)::value;
        const int key0 = t * TILE + 16 * g;
        uint32_t ex = (uint32_t)ve, nan = 0;                 // the lane's: tokens 4 (c & 3) .. of block c >> 2
        if (kMask) {                                         // a slot behind the last key may hold anything
            const int rest = p.s.keys - key0 - 4 * (c & 3);
            ex = rest >= 4 ? ex : rest <= 0 ? 0u : ex & ((1u << (8 * rest)) - 1u);
        }
        if (__builtin_amdgcn_ballot_w64(maybe_255(ex) != 0)) {               // rare
            const uint32_t m = bytes_255(ex);
            ex &= ~(m * 255u);                               // the value counts through its weight instead
            nan = ((m & 1u) | (m >> 7 & 2u) | (m >> 14 & 4u) | (m >> 21 & 8u)) << (4 * (c & 3));
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) nan |= (uint32_t)__shfl_xor((int)nan, o, 64);
        }
        b8 w[NB][2][3];
#pragma unroll
        for (int b = 0; b < NB; ++b) weigh<kMask>([&](int u) { return kr[u]; }, q[b], ke, key0, seen[b], nan, st[b], w[b]);
        const bool more = t + 1 < t1;
        if (more) load_k(t + 1);
        each<4>([&](auto b) {
            constexpr int kB = b;
            uint32_t e[4];
            each<4>([&](auto i) { e[i] = __float_as_uint(row_lane<4 * kB + i>(__uint_as_float(ex))); });
            each<2>([&](auto h) {
                b8 lower, upper;
                values_bf16((uint32_t)vr[b][2 * h], (uint32_t)vr[b][2 * h + 1], e[2 * h], e[2 * h + 1], lower, upper);
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int k = 2; k >= 0; --k) {
                        st[n].acc[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lower, w[n][h][k], st[n].acc[2 * b], 0, 0, 0);
                        st[n].acc[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(upper, w[n][h][k], st[n].acc[2 * b + 1], 0, 0, 0);
                    }
            });
        });
        if (more) load_v();
    };
    const int t_clear = max(min(t1, clear_keys / TILE), t0);
    for (int t = t0; t < t_clear; ++t) step(std::false_type{}, t);
    for (int t = t_clear; t < t1; ++t) step(std::true_type{}, t);

    // the four waves' states joined in LDS; a lone part writes the output
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const float l = rows_sum(st[b].l);
        if (g == 0) {
            s_m[wave][16 * b + c] = st[b].reference();
            s_l[wave][16 * b + c] = l;
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        if (16 * b >= n_cols) break;                         // uniform
        if (b > 0) __syncthreads();
        if (16 * b + c < n_cols)
#pragma unroll
            for (int d = 0; d < DB; ++d) *reinterpret_cast<f4*>(&s_acc[wave][c][16 * d + 4 * g]) = st[b].acc[d];
        __syncthreads();
        for (int e = tid; e < 16 * (HD / 4); e += THREADS) {
            const int cc = e / (HD / 4), d4 = e % (HD / 4), col = 16 * b + cc;
            if (col >= n_cols) continue;
            float m = s_m[0][col];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) m = fmaxf(m, s_m[w][col]);
            f4 sum = f4{0.f, 0.f, 0.f, 0.f};
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const Factor f(s_m[w][col] - m);
                sum += f * *reinterpret_cast<const f4*>(&s_acc[w][cc][4 * d4]);
                l += f * s_l[w][col];
            }
            if (p.parts == 1) {
                const int r = col / G, hh = col - r * G;
                const float n = p.s.keys > 0 ? 1.0f / l : 0.f;
                *reinterpret_cast<f4*>(a.o + ((int64_t)(p.s.row0 + r) * NH + kvh * G + hh) * HD + 4 * d4) = sum * n;
            } else {
                const int64_t at = ((int64_t)kvh * a.slots + slot) * COLS + col;
                *reinterpret_cast<f4*>(a.acc + at * HD + 4 * d4) = sum;
                if (d4 == 0) a.ml[at] = f2{m, l};
            }
        }
    }
}

// ---- many columns ----

// Each wave has its own 16 columns of a group, and all go over the same keys: V's
// conversion to bf16 is done once for 64 columns, and a tile's loads once.  Wave w brings
// page w of a tile through its registers to LDS: K's codes and exponents as they are (pages
// 64 B further apart than they are long, so that the operand reads are free of bank
// conflicts), V as bf16 in operand order, two tiles of everything.  A tile's loads go out
// at the start of the tile before it; one barrier per tile.
__global__ void __launch_bounds__(THREADS, 2) q4_many_kernel(AttnArgs a) {
    constexpr int COLS = kManyCols;
    constexpr int kPageLds = kQ4KBytes + 64, kStage = kTilePages * kPageLds;
    constexpr int kOut = 16 * kAccRow * 4;                   // a block's results, per wave
    constexpr int kVTile = 2 * DB * 1024;
    static_assert(kTilePages == WAVES, "a page per wave");
    static_assert(WAVES * kOut <= 2 * kStage + 2 * kVTile, "the results overwrite the tiles");
    __shared__ __attribute__((aligned(16))) unsigned char s_mem[2 * kStage + 2 * kVTile];
    __shared__ int s_ke[2][kTilePages][16];                  // K exponents
    __shared__ uint32_t s_nan[2][kTilePages];                // tokens whose value is NaN
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int g = lane >> 4, c = lane & 15;
    const int kvh = blockIdx.x, w = blockIdx.y;

    Place at, to;
    find_stretch(a, w, at, to);
    i4 piece[2] = {i4{-1, 0, 0, 0}, i4{-1, 0, 0, 0}};        // the group begun before this stretch; the one it leaves open
    for (;;) {
        if (at.sess >= a.n_sess || at.sess > to.sess ||
            (at.sess == to.sess && (at.group > to.group || (at.group == to.group && at.tile >= to.tile))))
            break;
        Session s = session_of<true>(a, at.sess);
        s = Session{__builtin_amdgcn_readfirstlane(s.keys), __builtin_amdgcn_readfirstlane(s.past),
                    __builtin_amdgcn_readfirstlane(s.rows), __builtin_amdgcn_readfirstlane(s.row0)};
        if (at.group >= n_groups(s)) {
            at = Place{at.sess + 1, 0, 0};
            continue;
        }
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

        // ---- a tile's way into LDS ----
        const int32_t* table = a.tables + sess * a.table_stride;
        const int last_page = (s.keys - 1) >> kKvBlockShift;
        int win = -64, held = 0;                             // 64 table entries from `win` on
        i4 kr, vr, ve;
        int ke = 0;
        auto load = [&](int t) {                             // page `wave` of tile t
            const int pg = t * kTilePages;
            if (pg + kTilePages > win + 64) {
                win = pg;
                held = table[min(pg + lane, last_page)];
            }
            const int e = __builtin_amdgcn_readlane(held, min(pg + wave, last_page) - win);
            const int phys = (unsigned)e < (unsigned)a.nb ? e : 0;           // an entry outside the pool reads page 0
            const uint8_t* rec = a.pool + phys * kQ4Page + kvh * kQ4Rec;
            kr = *reinterpret_cast<const i4*>(rec + 16 * lane);
            vr = *reinterpret_cast<const i4*>(rec + kQ4VOff + 16 * lane);
            ve = *reinterpret_cast<const i4*>(rec + kQ4VeOff + 16 * g);      // block g's exponents of the page's tokens
            ke = *reinterpret_cast<const int*>(rec + kQ4KeOff + 4 * c);
        };
        auto put = [&](int t) {                              // lane (g, c): dims 32 g + c and 32 g + 16 + c
            *reinterpret_cast<i4*>(s_mem + (t & 1) * kStage + wave * kPageLds + 16 * lane) = kr;
            if (lane < 16) s_ke[t & 1][wave][c] = ke;
            const int rest = s.keys - t * TILE - 16 * wave;  // a slot behind the last key may hold anything
            uint32_t nan = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t x = (uint32_t)ve[i];
                if (rest < 16) x = rest >= 4 * i + 4 ? x : rest <= 4 * i ? 0u : x & ((1u << (8 * (rest - 4 * i))) - 1u);
                nan |= maybe_255(x);
                ve[i] = (int)x;
            }
            if (__builtin_amdgcn_ballot_w64(nan != 0)) {     // rare
                nan = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t m = bytes_255((uint32_t)ve[i]);
                    ve[i] &= (int)~(m * 255u);               // the value counts through its weight instead
                    nan |= ((m & 1u) | (m >> 7 & 2u) | (m >> 14 & 4u) | (m >> 21 & 8u)) << (4 * i);
                }
                nan |= (uint32_t)__shfl_xor((int)nan, 16, 64);
                nan |= (uint32_t)__shfl_xor((int)nan, 32, 64);
            }
            if (lane == 0) s_nan[t & 1][wave] = nan;
            unsigned char* dst = s_mem + 2 * kStage + (t & 1) * kVTile + g * 4096 + (16 * wave + c) * 16;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                b8 lower, upper;
                values_bf16((uint32_t)vr[2 * h], (uint32_t)vr[2 * h + 1], (uint32_t)ve[2 * h], (uint32_t)ve[2 * h + 1], lower, upper);
                *reinterpret_cast<b8*>(dst + h * 1024) = lower;
                *reinterpret_cast<b8*>(dst + 2048 + h * 1024) = upper;
            }
        };
        load(t_lo);
        QTerms q;
        int seen;
        State st;
        load_q(a, s, kvh, col0 + c, q, seen);
        st.clear();
        put(t_lo);
        __syncthreads();
        const uint32_t k_off = (uint32_t)((c >> 2) * kPageLds + (c & 3) * 64 + g * 16);
        auto tile = [&](auto mask_tag, int t) {
            constexpr bool kMask = decltype(mask_tag)::value;
            const unsigned char* k_at = s_mem + (t & 1) * kStage + k_off;
            const unsigned char* v_at = s_mem + 2 * kStage + (t & 1) * kVTile + 16 * lane;
            b8 p[2][3];
            weigh<kMask>([&](int u) { return *reinterpret_cast<const i4*>(k_at + 256 * u); }, q, s_ke[t & 1][c >> 2][4 * (c & 3) + g],
                         t * TILE + 16 * g, seen, s_nan[t & 1][g], st, p);
#pragma unroll
            for (int d = 0; d < DB; d += 2) {                // two 16-dim blocks, two halves of their tokens
                b8 v[2][2];
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h) v[x][h] = *reinterpret_cast<const b8*>(v_at + 1024 * (2 * (d + x) + h));
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int k = 2; k >= 0; --k)
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            st.acc[d + x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[x][h], p[h][k], st.acc[d + x], 0, 0, 0);
            }
        };
        // every wave goes through all tiles of the stretch, for its page of them and the
        // barrier; its own columns need the first ones, up to t_clear without a mask
        auto round = [&](int t, auto&& compute) {
            if (t + 1 < t_hi) load(t + 1);
            compute();
            if (t + 1 < t_hi) put(t + 1);
            __syncthreads();
        };
        int t = t_lo;
        for (; t < min(t1, t_clear); ++t) round(t, [&] { tile(std::false_type{}, t); });
        for (; t < t1; ++t) round(t, [&] { tile(std::true_type{}, t); });
        for (; t < t_hi; ++t) round(t, [] {});

        // results through LDS (every wave is past its tiles), rows in address order:
        // the output, or a piece of a group that others have the rest of
        const bool whole = t_lo == 0 && t_hi == tiles;
        const int slot = 2 * w + (t_lo > 0 ? 0 : 1);
        if (!whole) piece[t_lo > 0 ? 0 : 1] = i4{sess, group, t_hi == tiles, min(n_cols - group * COLS, COLS)};
        unsigned char* mine = s_mem + wave * kOut;
        if (col0 < n_cols) {
            const float l = rows_sum(st.l), m = st.reference();
#pragma unroll
            for (int d = 0; d < DB; ++d) *reinterpret_cast<f4*>(mine + (c * kAccRow + 16 * d + 4 * g) * 4) = st.acc[d];
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
        __syncthreads();                                     // the next group's tiles come where the results were
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
    if constexpr (kCausal) {
        if (f.many) {
            hipLaunchKernelGGL(q4_many_kernel, dim3(NKV, a.gw), dim3(THREADS), 0, s, a);
            NOVA_LAUNCHED();
            hipLaunchKernelGGL(many_join_kernel, dim3(join_wgs), dim3(THREADS), 0, s, a);
            NOVA_LAUNCHED();
            return;
        }
    }
    // Tables this short: a workgroup per session and kv head, nothing to join.
    const bool solo = a.table_stride <= kSoloPages;
    if (solo) a.min_share = kSoloPages;
    const dim3 grid(NKV, solo ? a.n_sess : f.slots);
    // The pages of a pool larger than the 256 MB memory-side cache (all layers of it,
    // as a step walks through them) come from HBM.
    const bool once = (int64_t)Model::L * a.nb * kQ4Page > (int64_t)256 << 20;
    auto run = [&](auto once_tag) {
        constexpr bool kOnce = decltype(once_tag)::value;
        if (f.cols == 16) hipLaunchKernelGGL((q4_few_kernel<1, kCausal, kOnce>), grid, dim3(THREADS), 0, s, a);
        if constexpr (kCausal)
            if (f.cols == 32) hipLaunchKernelGGL((q4_few_kernel<2, true, kOnce>), grid, dim3(THREADS), 0, s, a);
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
