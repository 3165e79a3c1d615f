// attn_q8.hip -- attention over the 8-bit pages (kv_q8.h): one query token per
// session (decode), or a ragged chunk of new tokens per session, causally.
//
// o_h = sum_t softmax_t(q_h . k_t / sqrt(HD)) v_t, k_t = ks_t * code, v_t = vs_t * code,
// over keys [0, n_keys) or, for row r of a chunk, [0, n_past + r].
//
// Numbers.  The codes are exact operands: the query goes into three signed digits of
// base 256 against K's int8 codes (products and sums are exact integers), and a
// weight times V's scale into two fp16 terms against V's codes, which fp16 holds
// exactly; sums are fp32.  That costs one and a half fp16 products for the scores and
// two for the output, and rounds in two places where fp32 operations would not:
//   * the query to 2^-24 of its largest component.  A component far below that one
//     loses bits which count only where K is exactly 0 beside the large one (a
//     channel 1000 times the others: 3e-5); elsewhere the quantiser's half step, 2^-8
//     of the row's largest |k|, under the large component outweighs them by far;
//   * a weight times scale to 2^-30 of the row's largest one, so n keys that share a sum
//     with one that outweighs each of them by far lose at most n 2^-30 of it.
// With rows as projections give them the result is 7e-8 (a handful of keys) to 6.3e-7
// (tens of thousands) from 64 bits, where fp32 operations on the decoded values are
// 1e-7 to 2e-6.
//
// One pass over the keys with a running reference and sum of the softmax.  The
// reference m of the weights 2^(s - m) follows the largest weight times V scale, lazily:
// that product may drift from 2^kTop to 2^kLazy, which the two fp16 terms have room
// for, so that almost no tile rescales its sums (kTop 2 instead of 6: 3% off the
// 8 x 512 tokens below, and 4 bits off the small products).
//
// Two kernels, by the columns (query rows x heads of a kv head) that a session may
// have.  Up to 32: the waves of a workgroup share them and split the keys; K and V
// go from the pages to registers once and HBM bounds it.  8 x 32768 keys of the 14B
// model, 554 MB: 90 us, 6.2 TB/s; 16 sessions of 512 to 8192 keys (7B), 66 MB: 21.8 us
// in two launches.  Above: 64 columns a workgroup, K and V through LDS, the
// matrix instructions and the softmax's vector instructions bound it, of which a SIMD
// overlaps a part only (a 16x16x32 product and 4 vector instructions take 16 and 16
// clocks alone, 28 together).  8 x 512 tokens behind up to 4096 (7B), 122 GFLOP: 272 us, 450
// TFLOP/s of the result's own products, twice that with the digits and terms.  A wave with
// 32 columns, whose bigger products leave the vector unit more room, was 10 to 20%
// slower: its operands and sums fill the 256 registers of two waves per SIMD, and
// nothing is loaded ahead.  Three waves per SIMD, loads two tiles ahead and the scores of a tile
// under the products of the one before it came out within 2% or slower.
#include <hip/hip_runtime.h>
#include <cstdint>
#include <type_traits>

namespace nova {
namespace {
// Many columns, 12 prompts of up to 300 tokens (1.5B) / 8 x 512 tokens behind up to
// 4096 (7B), us.  Fewest tiles of a piece of a group: 2 37.3 / 266, 3 36.0 / 266, 4 39.0 / 272.
constexpr int kMinPiece = 3;
// What a group costs beside its tiles, in tiles: 0 43.2 / 277, 2 36.6 / 276, 4 39.0 / 272,
// 8 35.7 / 279 with pieces of 4; short sessions need it most (8 of 19 rows, 7B: 0 135, 2 17.6,
// 4 11.8, 8 12.0), as a workgroup is given several of them.
constexpr int kGroupTiles = 4;
}  // namespace
}  // namespace nova

#include "attn_ragged.h"
#include "check.h"
#include "kv_q8.h"
#include "model.h"
#include "nova_kernel.h"

namespace nova {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr int kSoloPages = 48;                  // tables that take one launch, see launch()
constexpr float kTop = 6.f, kLazy = 15.9f;      // log2 of a column's largest weight times value scale: where it is put, where it may drift
constexpr int kUnitLeast = -125, kUnitMost = 36;   // log2 of the units of value scales; 1 / unit is finite
constexpr float kFloor = -82.f, kUnitRoom = 0x1p86f;   // log2 of the smallest scale in units that the reference follows; the largest scale

// ---- operands ----

// A column's query in base 256: x = q / max|q| * 127 * 2^16 rounded to an integer,
// x = 65536 d[0] + 256 d[1] + d[2] with signed digits, which is q to 2^-23 of its
// largest component; int8 products against the K codes are exact, so a score
// has fp32's accuracy.  Lane (g, c) holds dims 64 h + 16 g .. + 15 of column c.
struct QDigits {
    i4 d[3][2];
    float scale;               // of an integer score, 1/sqrt(HD) and log2 e included
};

__device__ __forceinline__ void q_digits(const f4 (&x)[2][4], QDigits& out) {
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[h][j][e]) & 0x7fffffffu);
    // as floats the bits of NaN are lost, so the lanes are joined as integers
    auto s = __builtin_amdgcn_permlane16_swap(top, top, false, false);
    top = max((uint32_t)s[0], (uint32_t)s[1]);
    s = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    top = max((uint32_t)s[0], (uint32_t)s[1]);
    const bool finite = top < 0x7f800000u, live = finite && top > 0;
    int ex = 0;
    const float m = live ? frexpf(__uint_as_float(top), &ex) : 1.f;    // largest = m 2^ex, m in [1/2, 1)
    constexpr float kUnit = 127.f * 65536.f;
    // the factor in two steps, so that neither leaves fp32 (the first is a power of two)
    const float f0 = live ? ldexpf(1.f, min(max(-ex, -126), 126)) : 0.f, f1 = live ? ldexpf(kUnit / m, -ex - min(max(-ex, -126), 126)) : 0.f;
    out.scale = finite ? ldexpf(m * (kScale * kLog2e / kUnit), ex) : __builtin_nanf("");
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t y[4];                                   // digits plus 128 in bytes 2, 1, 0
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = finite ? x[h][j][e] * f0 * f1 : 0.f;
                y[e] = (uint32_t)((int)__builtin_rintf(v) + 0x808080);
            }
            // bytes of (y0, y1) and of (y2, y3) side by side, then the four of a digit
            const uint32_t a = __builtin_amdgcn_perm(y[1], y[0], 0x05010400u), b = __builtin_amdgcn_perm(y[3], y[2], 0x05010400u);
            const uint32_t c = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0602u), d = __builtin_amdgcn_perm(y[3], y[2], 0x0c0c0602u);
            out.d[0][h][j] = (int)(__builtin_amdgcn_perm(d, c, 0x05040100u) ^ 0x80808080u);
            out.d[1][h][j] = (int)(__builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u);
            out.d[2][h][j] = (int)(__builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u);
        }
}

// 8 int8 codes as fp16, exactly: 1024 + (c + 128) has the bits 0x6400 | (c + 128)
__device__ __forceinline__ h8 codes_f16(uint32_t w0, uint32_t w1) {
    u4 r;
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    r[0] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u);
    r[1] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u);
    r[2] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u);
    r[3] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u);
    return __builtin_bit_cast(h8, r) + (_Float16)-1152.0f;
}

// weights e in fp16 terms hi + lo (hi cut off, lo the rest: 21 bits, fewer below 2^-3, as lo ends at 2^-24)
__device__ __forceinline__ void split_f16(const float (&e)[8], h8& hi, h8& lo) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(e[j], e[j + 1]));
        const float r0 = __builtin_fmaf((float)h[0], -1.f, e[j]), r1 = __builtin_fmaf((float)h[1], -1.f, e[j + 1]);
        const h2 r = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(r0, r1));
        hi[j] = h[0];
        hi[j + 1] = h[1];
        lo[j] = r[0];
        lo[j + 1] = r[1];
    }
}

// The query rows of a block's column, lane (g, c) its dims 64 h + 16 g .. + 15.
__device__ __forceinline__ void load_q(const AttnArgs& a, const Session& s, int kvh, int col, QDigits& out, int& seen) {
    const bool real = col < s.rows * G;
    const int r = real ? col / G : 0, hh = real ? col - r * G : 0;
    const float* src = a.q + ((int64_t)(s.row0 + r) * NH + kvh * G + hh) * HD + 16 * ((threadIdx.x & 63) >> 4);
    f4 x[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[h][j] = *reinterpret_cast<const f4*>(src + 64 * h + 4 * j);
            if (!real) x[h][j] = f4{0.f, 0.f, 0.f, 0.f};
        }
    q_digits(x, out);
    seen = real ? min(s.past + r + 1, s.keys) : 0;
}

// A block's state over the keys seen so far: lane (g, c) holds the reference, its
// share of the sum and dims 16 d + 4 g .. + 3 of column c.  Weights are 2^(s - m).
// They meet V's codes as 2^(s - m) vs in two fp16 terms, which end at 2^-24, so the
// reference follows the largest of these products among the keys that the column
// sees, not the largest score: what a key may lose is 2^-30 of the largest one, whatever
// the scales of keys that are hidden or weigh nothing.  A score above `limit` may move
// the reference (a column's first one always does).  The limit counts with the largest
// scale so far, so a key whose scale is far above the others makes more tiles look: one of
// 2^20 times per session costs 8 x 512 tokens (7B) 9%, one of 16 times 2%, the decode nothing.
struct State {
    float m, l, limit;
    f4 acc[DB];
    __device__ __forceinline__ void clear() {
        m = l = 0.f;
        limit = -INFINITY;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = f4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ bool unset() const { return limit == -INFINITY; }
    __device__ __forceinline__ float reference() const { return unset() ? kUnset : m; }
    __device__ __forceinline__ void scale_acc(float f) {
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] *= f;
    }
};

// V's scales in units, so that weights (2^(kTop - log2 vs) for the largest product)
// stay near 1, where a score less its reference is exact to 2^-22, and inside fp32 with
// their tails.  The unit is a power of two: the size of the first tile's largest scale, 2^36 at
// most.  It serves scales of 2^-82 to 2^86 of its own size; a larger one moves it (to
// 2^36 at most).  So a column loses bits only where the products that count have scales
// 2^82 times smaller than others of the session, hidden ones included, and below 2^-46.
struct ValueUnit {
    int ex;                    // log2 of the unit
    float inv;                 // 1 / unit
    float most, cap;           // no scale so far is larger; its log2 in units, or kFloor
    __device__ __forceinline__ float unit() const { return ldexpf(1.f, ex); }
    __device__ __forceinline__ void clear() {
        ex = 0;
        inv = 1.f;
        most = 0.f;
        cap = kFloor;
    }
    // vs: scale of the lane's key, 0 where there is none; returns it in units
    template <int NB>
    __device__ __forceinline__ float take(float vs, State (&st)[NB]) {
        if (__builtin_amdgcn_ballot_w64(vs > most)) {        // rare
            const float top = wave_max(vs);                  // (a NaN does not count)
            if (most == 0.f || top * inv > kUnitRoom) {
                int to;
                (void)frexpf(top, &to);
                to = min(max(to, kUnitLeast), kUnitMost);
                // products keep their size: the reference goes down by as much as the
                // unit goes up, as far as the weights' sum has room for, the sums for the rest
                if (most > 0.f)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        int e;
                        (void)frexpf(rows_max(st[b].l), &e);
                        const int by = min(max(90 - e, 0), to - ex);
                        st[b].m -= (float)by;
                        st[b].l = ldexpf(st[b].l, by);
                        st[b].scale_acc(ldexpf(1.f, by - (to - ex)));
                    }
                ex = to;
                inv = ldexpf(1.f, -to);
            }
            most = 1.125f * top;                             // (so that few tiles come here)
            cap = fmaxf(__builtin_amdgcn_logf(most * inv), kFloor);
#pragma unroll
            for (int b = 0; b < NB; ++b) st[b].limit = st[b].unset() ? -INFINITY : kLazy - cap;
        }
        return vs * inv;
    }
};

// Scores, weights and sum of one tile and block.  k_op(u): K operand u = 2 kb + h
// (dims 64 h .. of key block kb), q_op(d, h): the query's; ks and vs: the K scale of
// the lane's key and its V scale in units, none above 2^cap; key0: first key of the
// lane's page.  The weights come out in two fp16 terms, so that V's codes can follow as they are.
template <bool kMask, class K, class Q>
__device__ __forceinline__ void weigh(K&& k_op, Q&& q_op, float q_scale, float ks, float vs, float cap, int key0, int seen, State& st,
                                      h8 (&hi)[2], h8 (&lo)[2]) {
    // The lowest digit's sum starts at the bits of 1.5 * 2^23, so that it is that
    // float plus the sum without a conversion; the middle one starts 1.5 * 2^23 / 256
    // lower, which takes it off again.
    const i4 kLow = i4{0x4b400000, 0x4b400000, 0x4b400000, 0x4b400000}, kMid = i4{-49152, -49152, -49152, -49152};
    float x[16];
    float top = -INFINITY;
    // row 4g + i of key block kb: token 4 kb + i of page g.  The matrix instructions
    // of a key block go out before the vector instructions of the one before it.
    each<4>([&](auto kb) {
        i4 z[3] = {i4{0, 0, 0, 0}, kMid, kLow};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const i4 k = k_op(2 * kb + h);
#pragma unroll
            for (int d = 0; d < 3; ++d) z[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, q_op(d, h), z[d], 0, 0, 0);
        }
        each<4>([&](auto i) {
            constexpr int e = i, j = 4 * kb + i;
            // the two scales first: the sum of codes times K's alone may pass fp32
            const float w = fmaf((float)((z[0][e] << 8) + z[1][e]), 256.f, __int_as_float(z[2][e]));
            x[j] = fmaf(w, row_lane<j>(ks) * q_scale, -st.m);
            if (kMask && key0 + j >= seen) x[j] = -INFINITY;
            top = fmaxf(top, x[j]);
        });
    });
    if (__builtin_amdgcn_ballot_w64(top > st.limit)) {
        // rare: a column's first keys, and a product that may be above 2^kLazy (it is
        // where its key has the largest scale so far), which puts the reference to where
        // the largest product is 2^kTop
        const float r = fmaxf(__builtin_amdgcn_logf(vs), kFloor);
        float t = -INFINITY;
        each<16>([&](auto j) { t = fmaxf(t, x[j] + row_lane<j>(r)); });
        const float col_top = rows_max(t);
        const bool first = st.unset(), moves = first ? col_top > -INFINITY : rows_max(top) > st.limit && col_top > kTop;
        const float by = moves ? col_top - kTop : 0.f;
        const Factor corr(first ? -INFINITY : -by);
        st.m += by;
        st.limit = moves ? kLazy - cap : st.limit;
        st.l = corr * st.l;
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] -= by;
        // scores of 2^23 and more leave no room for log2 vs beside them: the product stays
        // below its bound all the same (and a NaN is left as it is)
        if (__builtin_amdgcn_ballot_w64(!(fabsf(by) < 0x1p20f)))
            each<16>([&](auto j) {
                const float most = kLazy - row_lane<j>(r);
                x[j] = x[j] > most ? most : x[j];
            });
        st.scale_acc(corr.half * corr.half);                 // (in one unit: what this loses weighs nothing)
    }
    float e[2][8];
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    each<16>([&](auto j) {
        const float w = __builtin_amdgcn_exp2f(x[j]);
        sum[j / 4] += w;
        // (the cross-lane read is not for the lanes of one side of a branch)
        const float y = w * row_lane<j>(vs);
        e[j / 8][j % 8] = kMask && key0 + j >= seen ? 0.f : y;   // a hidden value may be NaN
    });
    st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    split_f16(e[0], hi[0], lo[0]);
    split_f16(e[1], hi[1], lo[1]);
}

// ---- few columns ----
//
// Up to 16 NB columns (query rows x heads of a kv head) of a session: the
// workgroup's waves share them and each takes its own keys, 64 at a time, so K and
// V are read once and bound everything.  The operands come straight from the
// pages; the next tile's K loads go out behind the scores, V's behind the
// products, into the registers that these have just read.  kOnce: non-temporal
// loads, for pools that no cache holds until the next step (see launch()).
template <int NB, bool kCausal, bool kOnce>
__global__ void __launch_bounds__(THREADS, NB == 1 ? 2 : 1) q8_few_kernel(AttnArgs a) {
    constexpr int COLS = 16 * NB;
    __shared__ __attribute__((aligned(16))) float s_acc[WAVES][16][kAccRow];
    __shared__ float s_m[WAVES][COLS], s_l[WAVES][COLS];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, c = lane & 15;
    const int kvh = blockIdx.x % NKV, slot = blockIdx.x / NKV;
    const Part p = find_part<kCausal>(a, slot);
    if (p.sess < 0) return;
    if (kvh == 0 && p.index == 0 && tid == 0) a.info[p.sess] = i4{slot, p.parts, p.s.rows, p.s.row0};
    const int n_cols = p.s.rows * G;
    // the part's tiles, and this wave's of them
    const int tiles = (p.s.keys + TILE - 1) / TILE;
    const int t_lo = (int)((int64_t)tiles * p.index / p.parts), t_hi = (int)((int64_t)tiles * (p.index + 1) / p.parts);
    const int t0 = t_lo + (t_hi - t_lo) * wave / WAVES, t1 = t_lo + (t_hi - t_lo) * (wave + 1) / WAVES;
    const int clear_keys = min(p.s.past + 1, p.s.keys);      // keys below: seen by all columns

    // lane (g, c) reads K rows of page c >> 2 and V columns and scales of page g
    Pages pages(a, p.sess, p.s.keys);
    const uint8_t *k_at = nullptr, *v_at = nullptr;
    i4 kr[8], vr[DB];
    float ks = 0.f, vs = 0.f;
    auto load_k = [&](int t) {
        const int pg = t * kTilePages;
        pages.reach(pg);
        const uint8_t* head = a.pool + kvh * kQ8Rec;
        k_at = head + pages[pg + (c >> 2)] * kQ8Page + g * 64 + (c & 3) * 16;
        v_at = head + pages[pg + g] * kQ8Page;
#pragma unroll
        for (int u = 0; u < 8; ++u) kr[u] = page_load<kOnce>(k_at + 256 * u);
        ks = *reinterpret_cast<const float*>(v_at + kQ8KsOff + 4 * c);
        vs = *reinterpret_cast<const float*>(v_at + kQ8VsOff + 4 * c);
    };
    auto load_v = [&] {
#pragma unroll
        for (int u = 0; u < DB; ++u) vr[u] = page_load<kOnce>(v_at + kQ8VOff + 256 * u + 16 * c);
    };
    if (t0 < t1) {
        load_k(t0);
        load_v();
    }
    QDigits q[NB];
    int seen[NB];              // keys that the column sees
    State st[NB];
    ValueUnit unit;
    unit.clear();
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        load_q(a, p.s, kvh, 16 * b + c, q[b], seen[b]);
        st[b].clear();
    }
    auto step = [&](auto mask_tag, int t) {
        constexpr bool kMask = decltype(mask_tag)::value;
        const int key0 = t * TILE + 16 * g;
        // (a key behind the last one may hold anything)
        const float sv = unit.take(!kMask || key0 + c < p.s.keys ? vs : 0.f, st);
        h8 hi[NB][2], lo[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
            weigh<kMask>([&](int u) { return kr[u]; }, [&](int d, int h) { return q[b].d[d][h]; }, q[b].scale, ks, sv, unit.cap, key0, seen[b], st[b],
                         hi[b], lo[b]);
        const bool more = t + 1 < t1;
        if (more) load_k(t + 1);
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const h8 v = codes_f16((uint32_t)vr[d][2 * u], (uint32_t)vr[d][2 * u + 1]);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    st[b].acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi[b][u], st[b].acc[d], 0, 0, 0);
                    st[b].acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo[b][u], st[b].acc[d], 0, 0, 0);
                }
            }
        if (more) load_v();
    };
    const int t_clear = max(min(t1, clear_keys / TILE), t0);
    for (int t = t0; t < t_clear; ++t) step(std::false_type{}, t);
    for (int t = t_clear; t < t1; ++t) step(std::true_type{}, t);

    // the four waves' states joined in LDS; a lone part writes the output
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const float l = rows_sum(st[b].l);
        st[b].scale_acc(unit.unit());
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

// LDS byte address of a __shared__ location
__device__ __forceinline__ uint32_t lds_addr(const unsigned char* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)p;
}

// 2 KiB from a wave-uniform address straight to LDS, 16 B per lane: bytes 16 lane of
// each half.  In inline asm so that the compiler's own counts do not see the loads
// (it would drain them before every LDS read): the pipeline below waits for them.
// m0 holds the LDS address; the statement saves and restores it, and the scalar
// copy of the base settles a base that a vector instruction wrote and is the wait
// state that m0 needs before an LDS load.
__device__ __forceinline__ void page_to_lds(const void* base, uint32_t lane16, uint32_t lds) {
    uint32_t saved;
    uint64_t from;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %4\n\ts_mov_b64 %1, %2\n\tglobal_load_lds_dwordx4 %3, %1\n\t"
        "s_mov_b32 m0, %5\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %6, %1\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved), "=&s"(from)
        : "s"(base), "v"(lane16), "s"(lds), "s"(lds + 1024u), "v"(lane16 + 1024u)
        : "memory");
}

// Each wave has its own 16 columns of a group, and all go over the same keys: V's
// conversion to fp16 is done once for 64 columns, and a tile's loads once.
// Wave w brings page w of a tile: K straight to LDS, the
// pages 64 B further apart than they are long so that the operand reads are free of
// bank conflicts; V and the scales through registers, the codes turned into fp16 in
// operand order, two tiles of everything.  A tile's loads go
// out at the start of the tile before it and are waited for at its end; one barrier
// per tile.
__global__ void __launch_bounds__(THREADS, 2) q8_many_kernel(AttnArgs a) {
    constexpr int COLS = kManyCols;
    constexpr int kPageLds = kQ8KBytes + 64, kStage = kTilePages * kPageLds;
    constexpr int kOut = 16 * kAccRow * 4;                   // a block's results, per wave
    constexpr int kVTile = 2 * DB * 1024;
    static_assert(kTilePages == WAVES, "a page per wave");
    static_assert(WAVES * kOut <= 2 * kStage + 2 * kVTile, "the results overwrite the tiles");
    __shared__ __attribute__((aligned(16))) unsigned char s_mem[2 * kStage + 2 * kVTile];
    __shared__ float s_scale[2][2][TILE];                    // K scale, V scale
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
        i4 vr[2];
        float scale = 0.f;
        auto load = [&](int t) {                             // page `wave` of tile t
            const int pg = t * kTilePages;
            if (pg + kTilePages > win + 64) {
                win = pg;
                held = table[min(pg + lane, last_page)];
            }
            const int e = __builtin_amdgcn_readlane(held, min(pg + wave, last_page) - win);
            const int phys = (unsigned)e < (unsigned)a.nb ? e : 0;           // an entry outside the pool reads page 0
            const uint8_t* rec = a.pool + phys * kQ8Page + kvh * kQ8Rec;
#pragma unroll
            for (int u = 0; u < 2; ++u) vr[u] = *reinterpret_cast<const i4*>(rec + kQ8VOff + 1024 * u + 16 * lane);
            scale = *reinterpret_cast<const float*>(rec + kQ8KsOff + 4 * (lane & 31));
            page_to_lds(rec, 16 * lane, __builtin_amdgcn_readfirstlane(lds_addr(s_mem) + (t & 1) * kStage + wave * kPageLds));
        };
        auto put = [&](int t) {                              // waits for every load of the wave
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            unsigned char* dst = s_mem + 2 * kStage + (t & 1) * kVTile + g * 2048 + (16 * wave + c) * 16;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 2; ++e)                  // dims 64 u + 16 g + c, tokens 8 e .. + 7
                    *reinterpret_cast<h8*>(dst + u * 8192 + e * 1024) = codes_f16((uint32_t)vr[u][2 * e], (uint32_t)vr[u][2 * e + 1]);
            // (a key behind the last one may hold anything: its V scale is none)
            if (lane >= 16 && t * TILE + 16 * wave + c >= s.keys) scale = 0.f;
            if (lane < 32) s_scale[t & 1][lane >> 4][16 * wave + c] = scale;
        };
        // the workgroup's LDS writes are done; loads in flight stay there
        auto barrier = [&] {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        load(t_lo);
        QDigits q;
        int seen;
        State st[1];
        load_q(a, s, kvh, col0 + c, q, seen);
        st[0].clear();
        put(t_lo);
        barrier();
        ValueUnit unit;
        unit.clear();
        const uint32_t k_off = (uint32_t)((c >> 2) * kPageLds + g * 64 + (c & 3) * 16);
        auto tile = [&](auto mask_tag, int t) {
            constexpr bool kMask = decltype(mask_tag)::value;
            const int key0 = t * TILE + 16 * g;
            const unsigned char* k_at = s_mem + (t & 1) * kStage + k_off;
            const unsigned char* v_at = s_mem + 2 * kStage + (t & 1) * kVTile + 16 * lane;
            const float ks = s_scale[t & 1][0][lane], vs = unit.take(s_scale[t & 1][1][lane], st);
            h8 hi[2], lo[2];
            weigh<kMask>([&](int u) { return *reinterpret_cast<const i4*>(k_at + 256 * u); },
                         [&](int d, int h) { return q.d[d][h]; }, q.scale, ks, vs, unit.cap, key0, seen, st[0], hi, lo);
#pragma unroll
            for (int e = 0; e < 2 * DB / 4; ++e) {           // two 16-dim blocks, two halves of their tokens
                h8 v[2][2];
#pragma unroll
                for (int d = 0; d < 2; ++d)
#pragma unroll
                    for (int u = 0; u < 2; ++u) v[d][u] = *reinterpret_cast<const h8*>(v_at + 1024 * (2 * (2 * e + d) + u));
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            f4& o = st[0].acc[2 * e + d];
                            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[d][u], k ? lo[u] : hi[u], o, 0, 0, 0);
                        }
            }
        };
        // every wave goes through all tiles of the stretch, for its page of them and the
        // barrier; its own columns need the first ones, up to t_clear without a mask
        auto round = [&](int t, auto&& compute) {
            if (t + 1 < t_hi) load(t + 1);
            compute();
            if (t + 1 < t_hi) put(t + 1);
            barrier();
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
            const float l = rows_sum(st[0].l), m = st[0].reference();
            st[0].scale_acc(unit.unit());
#pragma unroll
            for (int d = 0; d < DB; ++d) *reinterpret_cast<f4*>(mine + (c * kAccRow + 16 * d + 4 * g) * 4) = st[0].acc[d];
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
    if constexpr (kCausal) {
        if (f.many) {
            hipLaunchKernelGGL(q8_many_kernel, dim3(NKV, a.gw), dim3(THREADS), 0, s, a);
            NOVA_LAUNCHED();
            hipLaunchKernelGGL(many_join_kernel, dim3(join_wgs), dim3(THREADS), 0, s, a);
            NOVA_LAUNCHED();
            return;
        }
    }
    // Tables this short: a workgroup per session and kv head, nothing to join (24
    // sessions of up to 600 keys, 7B: 9.6 us instead of 10.7 in two launches).
    const bool solo = a.table_stride <= kSoloPages;
    if (solo) a.min_share = kSoloPages;
    const dim3 grid((unsigned)(NKV * (solo ? a.n_sess : f.slots)));          // (slots may pass what a second dimension holds)
    // The pages of a pool larger than the 256 MB memory-side cache (all layers of it,
    // as a step walks through them) come from HBM: non-temporal loads, 8 x 32768 keys
    // of the 14B model 103 -> 90 us, 16 ragged sessions of the 7B model whose pages
    // are in no cache 23.7 -> 22.6.  Where a cache still has them plain loads are
    // faster: the same 16 sessions 20.7 instead of 22.0.
    const bool once = (int64_t)Model::L * a.nb * kQ8Page > (int64_t)256 << 20;
    auto run = [&](auto once_tag) {
        constexpr bool kOnce = decltype(once_tag)::value;
        if (f.cols == 16) hipLaunchKernelGGL((q8_few_kernel<1, kCausal, kOnce>), grid, dim3(THREADS), 0, s, a);
        if constexpr (kCausal)
            if (f.cols == 32) hipLaunchKernelGGL((q8_few_kernel<2, true, kOnce>), grid, dim3(THREADS), 0, s, a);
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

size_t attn_decode_q8_workspace_bytes(int n_sess) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535);
    return layout(shape(n_sess, 1), n_sess).total;
}

size_t attn_chunk_q8_workspace_bytes(int n_sess, int n_rows, int max_q) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && n_rows >= 0 && max_q >= 0 && max_q <= n_rows);
    return layout(shape(n_sess, max_q), n_sess).total;
}

void launch_attn_decode_q8_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                 const int32_t* n_keys, int n_sess, int layer, int nb, float* o, void* workspace,
                                 nova_stream_t s) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535);
    AttnArgs a = attn_args(kQ8Page, q, pool, tables, table_stride, n_keys, n_sess, layer, nb, o);
    NOVA_REQUIRE(workspace && aligned16(workspace));
    a.rows = RaggedRows{nullptr, 1, n_sess};
    a.max_q = 1;
    launch<false>(a, workspace, reinterpret_cast<hipStream_t>(s));
}

void launch_attn_chunk_q8_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                const int32_t* n_past, const int32_t* row_off, int n_sess, int n_rows, int max_q,
                                int layer, int nb, float* o, void* workspace, nova_stream_t s) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && n_rows >= 0 && n_rows <= (1 << 24));
    NOVA_REQUIRE(max_q >= 0 && max_q <= n_rows);
    NOVA_REQUIRE(row_off || n_rows % n_sess == 0);
    AttnArgs a = attn_args(kQ8Page, q, pool, tables, table_stride, n_past, n_sess, layer, nb, o);
    NOVA_REQUIRE(workspace && aligned16(workspace));
    if (n_rows == 0 || max_q == 0) return;
    a.rows = RaggedRows{row_off, n_rows / n_sess, n_rows};
    a.max_q = max_q;
    launch<true>(a, workspace, reinterpret_cast<hipStream_t>(s));
}

}  // extern "C"
