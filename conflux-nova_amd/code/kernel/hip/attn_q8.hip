// attn_q8.hip -- attention over the 8-bit pages (kv_q8.h): one query token per
// session (decode), or a ragged chunk of new tokens per session, causally.
//
// o_h = sum_t softmax_t(q_h . k_t / sqrt(HD)) v_t, k_t = ks_t * code, v_t = vs_t * code,
// over keys [0, n_keys) or, for row r of a chunk, [0, n_past + r].
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdint>
#include <type_traits>
#include <utility>

#include "check.h"
#include "kv_q8.h"
#include "model.h"
#include "nova_kernel.h"

namespace nova {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int NH = Model::NH, NKV = Model::NKV, HD = Model::HD, G = Model::G;
constexpr float kLog2e = 1.4426950408889634f;
#ifndef Q8_WPS
#define Q8_WPS (NB == 1 || kWide ? 2 : 1)
#endif
constexpr int WAVES = 4;
constexpr int THREADS = 64 * WAVES;
constexpr int TILE = 64;                       // keys of a wave's step: four pages
constexpr int kTilePages = TILE / kKvBlock;
constexpr int DB = HD / 16;                    // 16-dim blocks of the output
constexpr float kUnset = -1e30f;               // reference of a column without keys, where states are joined
constexpr float kTop = 6.f, kLazy = 14.f;      // log2 of a column's largest weight: where it is put, where it may drift
constexpr int kAccRow = HD + 4;                // floats per column in LDS: rows on different banks
static_assert(HD == 128 && kTilePages == 4 && G <= 16, "tile layout");

struct Q8Args {
    const float* q;            // [n_rows][NH][HD]
    const uint8_t* pool;       // the layer's first page
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* n_keys;     // decode: keys of each session; chunk: its prefix
    Q8Rows rows;
    int max_q;
    int n_sess;
    int nb;
    int gw;                    // workgroups aimed at per kv head
    int min_share;             // fewest tiles of a workgroup that shares a session
    int slots;                 // workgroups launched per kv head
    float* o;
    i4* info;                  // [n_sess] {first slot, parts, rows, first row}
    f2* ml;                    // [NKV][slots][cols] {reference, sum}
    float* acc;                // [NKV][slots][cols][HD]
};

// ---- small cross-lane helpers ----

// sum over lanes 0..l
__device__ __forceinline__ int scan_incl(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row 0 -> 1, 2 -> 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // rows 0, 1 -> 2, 3
    return v;
}

// lane N of each row of 16
template <int N>
__device__ __forceinline__ float row_lane(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x150 + N, 0xf, 0xf, true));
}

// over lanes c, c + 16, c + 32, c + 48
__device__ __forceinline__ float rows_max(float v) {
    auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
    auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}

template <int... I, class F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
    each_of(std::make_integer_sequence<int, N>{}, f);
}

// a wave's lanes have what its other lanes wrote to LDS
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ---- work split ----

// A session's rows (from row0 of the flat arrays), the keys its call attends to,
// and `past`: row r sees keys up to past + r (the decode's one row: up to past).
// Keys behind the session's table are left out.
struct Session {
    int keys, past, rows, row0;
};
template <bool kCausal>
__device__ __forceinline__ Session session_of(const Q8Args& a, int i) {
    Session s;
    s.rows = min(q8_count(a.rows, i), a.max_q);
    s.row0 = q8_row0(a.rows, i);
    const int n = max(a.n_keys[i], 0);
    const int64_t most = a.table_stride * kKvBlock, all = (int64_t)n + (kCausal ? s.rows : 0);
    s.keys = (int)(all < most ? all : most);
    s.past = kCausal ? n : s.keys - 1;
    return s;
}

struct Part {
    int sess;                  // < 0: nothing to do
    int index, parts;          // part `index` of `parts` of a column group's keys
    int group;                 // column group of the session
    int slot0;                 // the session's first slot
    Session s;
};

// columns of a workgroup: in the wide form each wave has its own
template <int NB, bool kWide>
constexpr int kGroupCols = 16 * NB * (kWide ? WAVES : 1);

// The session, column group and part of a slot.  A session has
// ceil(rows * G / cols) column groups, which its t tiles cost each; with T tiles in
// all and gw workgroups aimed at, each group is cut into ceil(t / share) parts,
// share = max(ceil(T / gw), min_share), so that no workgroup has more than a share
// whatever the lengths, and at most gw + (number of groups) slots are used.  Every
// wave works it out for itself, 64 sessions at a time.  The wide form, whose
// workgroups are few and long, takes the sessions with the most keys first and a
// session's last group, which sees the most of them, before its others, so that
// the short ones fill the end.
template <bool kCausal, int kCols, bool kSort>
__device__ __forceinline__ Part find_part(const Q8Args& a, int slot) {
    const int lane = threadIdx.x & 63;
    Session s{0, 0, 0, 0};
    int tiles = 0, groups = 0, index = lane;
    auto load = [&](int base) {
        s = Session{0, 0, 0, 0};
        if (base + lane < a.n_sess) s = session_of<kCausal>(a, base + lane);
        if constexpr (kSort) {
            const int n = min(a.n_sess - base, 64);
            int rank = lane < n ? 0 : lane;
            for (int j = 0; j < n; ++j) {
                const int k = __builtin_amdgcn_readlane(s.keys, j);
                if (lane < n) rank += k > s.keys || (k == s.keys && j < lane);
            }
            s.keys = __builtin_amdgcn_ds_permute(4 * rank, s.keys);
            s.past = __builtin_amdgcn_ds_permute(4 * rank, s.past);
            s.rows = __builtin_amdgcn_ds_permute(4 * rank, s.rows);
            s.row0 = __builtin_amdgcn_ds_permute(4 * rank, s.row0);
            index = __builtin_amdgcn_ds_permute(4 * rank, lane);
        }
        tiles = (s.keys + TILE - 1) / TILE;
        groups = (s.rows * G + kCols - 1) / kCols;
    };
    int total = 0;
    for (int base = 0; base < a.n_sess; base += 64) {
        load(base);
        total += __builtin_amdgcn_readlane(scan_incl(tiles * groups), 63);
    }
    const int share = max((total + a.gw - 1) / a.gw, a.min_share);
    int before = 0;
    for (int base = 0; base < a.n_sess; base += 64) {
        if (a.n_sess > 64) load(base);
        const int parts = max((tiles + share - 1) / share, 1);
        const int incl = before + scan_incl(parts * groups);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(incl > slot);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            Part p;
            p.sess = base + __builtin_amdgcn_readlane(index, l);
            p.parts = __builtin_amdgcn_readlane(parts, l);
            const int n_groups = __builtin_amdgcn_readlane(groups, l);
            p.slot0 = __builtin_amdgcn_readlane(incl, l) - p.parts * n_groups;
            const int e = slot - p.slot0;
            p.group = n_groups - 1 - e / p.parts;
            p.index = e % p.parts;
            p.s.keys = __builtin_amdgcn_readlane(s.keys, l);
            p.s.past = __builtin_amdgcn_readlane(s.past, l);
            p.s.rows = __builtin_amdgcn_readlane(s.rows, l);
            p.s.row0 = __builtin_amdgcn_readlane(s.row0, l);
            return p;
        }
        before = __builtin_amdgcn_readlane(incl, 63);
    }
    return Part{-1, 0, 0, 0, 0, {0, 0, 0, 0}};
}

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
    const float f = kUnit / m;
    out.scale = finite ? ldexpf(m * (kScale * kLog2e / kUnit), ex) : __builtin_nanf("");
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = live ? ldexpf(x[h][j][e], -ex) * f : 0.f;
                y[e] = (uint32_t)((int)__builtin_rintf(v) + 0x808080);   // digits plus 128
            }
            // byte 2, 1, 0 of the four integers, 128 taken off again
#pragma unroll
            for (int d = 0; d < 3; ++d) {
                const int sh = 16 - 8 * d;
                const uint32_t w = ((y[0] >> sh) & 255) | ((y[1] >> sh) & 255) << 8 | ((y[2] >> sh) & 255) << 16 |
                                   ((y[3] >> sh) & 255) << 24;
                out.d[d][h][j] = (int)(w ^ 0x80808080u);
            }
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

// weights e in fp16 terms hi + lo (hi cut off, lo the rest: 21 bits or more)
__device__ __forceinline__ void split_f16(const float (&e)[8], h8& hi, h8& lo) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const h2 h = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(e[j], e[j + 1]));
        const h2 r = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(e[j] - (float)h[0], e[j + 1] - (float)h[1]));
        hi[j] = h[0];
        hi[j + 1] = h[1];
        lo[j] = r[0];
        lo[j + 1] = r[1];
    }
}

// ---- the kernel ----
//
// A wave has NB blocks of 16 columns (query rows x heads of a kv head) and takes
// 64 keys at a time.  Few columns (!kWide): the workgroup's waves share the
// session's columns and each takes its own keys, so K and V are read once and
// bound everything.  Many columns (kWide): each wave has its own 16 NB columns and
// all go over the same keys.
template <int NB, bool kCausal, bool kWide>
__global__ void __launch_bounds__(THREADS, Q8_WPS) q8_attn_kernel(Q8Args a) {
    constexpr int COLS = kGroupCols<NB, kWide>;
    // in the wide form the query's digits stay in LDS, 1 KiB per operand, which the
    // results overwrite at the end; otherwise they stay in registers
    constexpr int kQOps = 6 * NB;
    constexpr int kWaveLds = kWide && kQOps * 1024 > 16 * kAccRow * 4 ? kQOps * 1024 : 16 * kAccRow * 4;
    __shared__ __attribute__((aligned(16))) unsigned char s_wave[WAVES][kWaveLds];
    __shared__ float s_m[WAVES][16 * NB], s_l[WAVES][16 * NB];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, g = lane >> 4, c = lane & 15;
    auto s_acc = [&](int w, int col, int d) { return reinterpret_cast<f4*>(s_wave[w] + (col * kAccRow + d) * 4); };
    const int kvh = blockIdx.x, slot = blockIdx.y;
    const Part p = find_part<kCausal, COLS, kWide>(a, slot);
    if (p.sess < 0) return;
    if (kvh == 0 && slot == p.slot0 && tid == 0) a.info[p.sess] = i4{p.slot0, p.parts, p.s.rows, p.s.row0};
    const int n_cols = p.s.rows * G;
    const int col0 = kWide ? p.group * COLS + wave * 16 * NB : 0;            // this wave's columns
    // the group's tiles, the part's of them, and this wave's of those
    const int group_keys = kCausal && kWide ? min(p.s.past + min(p.group * COLS + COLS - 1, n_cols - 1) / G + 1, p.s.keys) : p.s.keys;
    const int tiles = (group_keys + TILE - 1) / TILE;
    const int t_lo = (int)((int64_t)tiles * p.index / p.parts), t_hi = (int)((int64_t)tiles * (p.index + 1) / p.parts);
    int t0 = t_lo, t1 = t_hi;
    if constexpr (kWide) {
        const int wave_keys = min(p.s.past + min(col0 + 16 * NB - 1, n_cols - 1) / G + 1, p.s.keys);
        t1 = col0 < n_cols ? min(t_hi, (wave_keys + TILE - 1) / TILE) : t_lo;
    } else {
        t0 = t_lo + (t_hi - t_lo) * wave / WAVES;
        t1 = t_lo + (t_hi - t_lo) * (wave + 1) / WAVES;
    }
    const int clear_keys = min(p.s.past + col0 / G + 1, p.s.keys);             // keys below: seen by all of the wave's columns
    const int32_t* table = a.tables + p.sess * a.table_stride;
    const int last_page = (p.s.keys - 1) >> kKvBlockShift;

    // Pages of a tile: lane (g, c) reads K rows of page c >> 2 and V columns and
    // scales of page g.  64 table entries at a time stay in a register.
    int win = -64, win_pages = 0;
    auto phys = [&](int pg) {                                // pg: per lane, within the window
        const int v = __shfl(win_pages, min(pg, last_page) - win, 64);
        return (unsigned)v < (unsigned)a.nb ? v : 0;
    };
    const uint8_t* k_at;
    const uint8_t* v_at;
    auto locate = [&](int t) {
        const int pg = t * kTilePages;
        if (pg + kTilePages > win + 64) {                    // uniform
            win = pg;
            win_pages = table[min(pg + lane, last_page)];
        }
        const uint8_t* head = a.pool + kvh * kQ8Rec;
        k_at = head + phys(pg + (c >> 2)) * kQ8Page + g * 64 + (c & 3) * 16;
        v_at = head + phys(pg + g) * kQ8Page;
    };
    i4 kr[8], vr[DB];
    float ks, vs;
    auto load_k = [&] {
#pragma unroll
        for (int u = 0; u < 8; ++u) kr[u] = *reinterpret_cast<const i4*>(k_at + 256 * u);
        ks = *reinterpret_cast<const float*>(v_at + kQ8KsOff + 4 * c);
    };
    auto load_v = [&] {
        vs = *reinterpret_cast<const float*>(v_at + kQ8VsOff + 4 * c);
#pragma unroll
        for (int u = 0; u < DB; ++u) vr[u] = *reinterpret_cast<const i4*>(v_at + kQ8VOff + 256 * u + 16 * c);
    };
    if (t0 < t1) {
        locate(t0);
        load_k();
        load_v();
    }

    QDigits q[NB];
    int seen[NB];              // keys that the column sees
    // running reference and sum of the column; a score above `limit` moves the reference
    float m[NB], l[NB], limit[NB];
    f4 acc[NB][DB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int col = col0 + 16 * b + c;
        const bool real = col < n_cols;
        const int r = real ? col / G : 0, hh = real ? col - r * G : 0;
        const float* src = a.q + ((int64_t)(p.s.row0 + r) * NH + kvh * G + hh) * HD + 16 * g;
        f4 x[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[h][j] = *reinterpret_cast<const f4*>(src + 64 * h + 4 * j);
                if (!real) x[h][j] = f4{0.f, 0.f, 0.f, 0.f};
            }
        q_digits(x, q[b]);
        if constexpr (kWide)
#pragma unroll
            for (int e = 0; e < 6; ++e)
                *reinterpret_cast<i4*>(s_wave[wave] + (6 * b + e) * 1024 + 16 * lane) = q[b].d[e / 2][e % 2];
        seen[b] = real ? min(p.s.past + r + 1, p.s.keys) : 0;
        m[b] = l[b] = 0.f;
        limit[b] = -INFINITY;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[b][d] = f4{0.f, 0.f, 0.f, 0.f};
    }

    auto q_op = [&](int b, int d, int h) -> i4 {
        if constexpr (kWide) return *reinterpret_cast<const i4*>(s_wave[wave] + (6 * b + 2 * d + h) * 1024 + 16 * lane);
        else return q[b].d[d][h];
    };
    // The lowest digit's sum starts at the bits of 1.5 * 2^23, so that it is that
    // float plus the sum without a conversion; the middle one starts 1.5 * 2^23 / 256
    // lower, which takes it off again.
    const i4 kLow = i4{0x4b400000, 0x4b400000, 0x4b400000, 0x4b400000}, kMid = i4{-49152, -49152, -49152, -49152};
    auto step = [&](auto mask_tag, int t) {
        constexpr bool kMask = decltype(mask_tag)::value;
        if constexpr (kWide) asm volatile("" ::: "memory");  // the digits are read anew, not kept in 48 registers
        const int key0 = t * TILE + 16 * g;
        // lane (g, c) has the scales of token c of page g; a key behind the last
        // one may hold anything
        float sv = vs == 0.f ? 0x1p-20f : vs;
        if (kMask && key0 + c >= p.s.keys) sv = 1.f;
        const float lv = __builtin_amdgcn_logf(sv), inv = __builtin_amdgcn_rcpf(sv);
        h8 hi[NB][2], lo[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            // scores: key block kb has row 4g + i = token 4 kb + i of page g
            float x[16];
            float top = -INFINITY;
            each<4>([&](auto kb) {
                i4 z[3] = {i4{0, 0, 0, 0}, kMid, kLow};
#pragma unroll
                for (int d = 0; d < 3; ++d)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        z[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[2 * kb + h], q_op(b, d, h), z[d], 0, 0, 0);
                each<4>([&](auto i) {
                    constexpr int e = i, j = 4 * kb + i;
                    const float w = fmaf((float)((z[0][e] << 8) + z[1][e]), 256.f, __int_as_float(z[2][e])) * row_lane<j>(ks);
                    x[j] = fmaf(w, q[b].scale, row_lane<j>(lv) - m[b]);
                    if (kMask && key0 + j >= seen[b]) x[j] = -INFINITY;
                    top = fmaxf(top, x[j]);
                });
            });
            if (__builtin_amdgcn_ballot_w64(top > limit[b])) {
                // rare: a column's first keys, and a score more than kLazy above the
                // reference, put it to kTop below the largest score
                const float col_top = rows_max(top);
                const bool moves = col_top > limit[b];
                const float by = moves ? col_top - kTop : 0.f;
                const float corr = limit[b] == kLazy ? __builtin_amdgcn_exp2f(-by) : 0.f;
                m[b] += by;
                limit[b] = moves ? kLazy : limit[b];
                l[b] *= corr;
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] -= by;
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[b][d] *= corr;
            }
            float e[2][8];
            each<16>([&](auto j) {
                const float w = __builtin_amdgcn_exp2f(x[j]);
                e[j / 8][j % 8] = w;
                // (the cross-lane read is not for the lanes of one side of a branch)
                const float share = row_lane<j>(inv) * w;
                if (kMask) l[b] += key0 + j >= seen[b] ? 0.f : share;
                else l[b] += share;
            });
            split_f16(e[0], hi[b][0], lo[b][0]);
            split_f16(e[1], hi[b][1], lo[b][1]);
        }
        const bool more = t + 1 < t1;
        if (more) {
            locate(t + 1);
            load_k();
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const h8 v = codes_f16((uint32_t)vr[d][2 * u], (uint32_t)vr[d][2 * u + 1]);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    acc[b][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi[b][u], acc[b][d], 0, 0, 0);
                    acc[b][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo[b][u], acc[b][d], 0, 0, 0);
                }
            }
        if (more) load_v();
    };
    const int t_clear = max(min(t1, clear_keys / TILE), t0);
    for (int t = t0; t < t_clear; ++t) step(std::false_type{}, t);
    for (int t = t_clear; t < t1; ++t) step(std::true_type{}, t);

    // ---- the waves' results through LDS: each wave's own columns, or the four
    // states of the same columns joined; a lone part writes the output ----
    const bool lone = p.parts == 1;
    auto put = [&](int col, int d4, f4 sum, float mm, float ll) {            // col of the session
        if (lone) {
            const int r = col / G, hh = col - r * G;
            const float n = p.s.keys > 0 ? 1.0f / ll : 0.f;
            *reinterpret_cast<f4*>(a.o + ((int64_t)(p.s.row0 + r) * NH + kvh * G + hh) * HD + 4 * d4) = sum * n;
        } else {
            const int64_t at = ((int64_t)kvh * a.slots + slot) * COLS + col - p.group * COLS;
            *reinterpret_cast<f4*>(a.acc + at * HD + 4 * d4) = sum;
            if (d4 == 0) a.ml[at] = f2{mm, ll};
        }
    };
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        l[b] = rows_sum(l[b]);
        if (g == 0) {
            s_m[wave][16 * b + c] = limit[b] == kLazy ? m[b] : kUnset;
            s_l[wave][16 * b + c] = l[b];
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        if (col0 + 16 * b >= n_cols) break;                  // the same for all waves unless kWide
        if (b > 0 && !kWide) __syncthreads();
        if (col0 + 16 * b + c < n_cols)
#pragma unroll
            for (int d = 0; d < DB; ++d) *s_acc(wave, c, 16 * d + 4 * g) = acc[b][d];
        if constexpr (kWide) {
            wave_lds_sync();
#pragma unroll
            for (int e = lane; e < 16 * (HD / 4); e += 64) {
                const int cc = e / (HD / 4), d4 = e % (HD / 4), col = col0 + 16 * b + cc;
                if (col < n_cols)
                    put(col, d4, *s_acc(wave, cc, 4 * d4), s_m[wave][16 * b + cc],
                        s_l[wave][16 * b + cc]);
            }
            wave_lds_sync();
            continue;
        }
        __syncthreads();
        for (int e = tid; e < 16 * (HD / 4); e += THREADS) {
            const int cc = e / (HD / 4), d4 = e % (HD / 4), col = 16 * b + cc;
            if (col >= n_cols) continue;
            float mm = s_m[0][col];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) mm = fmaxf(mm, s_m[w][col]);
            f4 sum = f4{0.f, 0.f, 0.f, 0.f};
            float ll = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float f = __builtin_amdgcn_exp2f(s_m[w][col] - mm);
                sum += *s_acc(w, cc, 4 * d4) * f;
                ll += s_l[w][col] * f;
            }
            put(col, d4, sum, mm, ll);
        }
    }
}

// Joins the parts of the sessions that were cut.  Columns of all kv heads are
// dealt out over the grid: a workgroup each, its waves taking every fourth part
// (few columns, up to many parts), or a wave each (kWide: many columns).
template <bool kWide>
__global__ void __launch_bounds__(THREADS) q8_join_kernel(Q8Args a, int cols) {
    __shared__ f2 s_o[WAVES][64];
    __shared__ float s_l[WAVES], s_m[WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int first = kWide ? blockIdx.x * WAVES + wave : blockIdx.x, stride = kWide ? gridDim.x * WAVES : gridDim.x;
    int64_t done = 0;                                        // columns of the sessions before this batch of 64
    for (int base = 0; base < a.n_sess; base += 64) {
        i4 in = i4{0, 0, 0, 0};
        if (base + lane < a.n_sess && q8_count(a.rows, base + lane) > 0) in = a.info[base + lane];
        const int mine = in[1] > 1 ? in[2] * NH : 0;
        const int incl = scan_incl(mine);
        const int all = __builtin_amdgcn_readlane(incl, 63);
        int u = (int)((first + stride - done % stride) % stride);
        for (; u < all; u += stride) {                       // uniform over the workgroup unless kWide
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > u));
            const int e = u - (__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(mine, l));
            const int slot0 = __builtin_amdgcn_readlane(in[0], l), parts = __builtin_amdgcn_readlane(in[1], l);
            const int n_cols = __builtin_amdgcn_readlane(in[2], l) * G, row0 = __builtin_amdgcn_readlane(in[3], l);
            const int kvh = e / n_cols, col = e % n_cols;
            const int at = slot0 + ((n_cols - 1) / cols - col / cols) * parts;
            if (at + parts > a.slots) continue;              // offsets that do not add up: more groups than rows allow
            const int64_t from = ((int64_t)kvh * a.slots + at) * cols + col % cols;
            float m = kUnset, ll = 0.f;
            f2 o = f2{0.f, 0.f};
            for (int p = kWide ? 0 : wave; p < parts; p += kWide ? 1 : WAVES) {
                const f2 x = a.ml[from + (int64_t)p * cols];
                const f2 v = *reinterpret_cast<const f2*>(a.acc + (from + (int64_t)p * cols) * HD + 2 * lane);
                const float to = fmaxf(m, x[0]);
                const float f0 = __builtin_amdgcn_exp2f(m - to), f1 = __builtin_amdgcn_exp2f(x[0] - to);
                ll = ll * f0 + x[1] * f1;
                o = o * f0 + v * f1;
                m = to;
            }
            if constexpr (!kWide) {
                __syncthreads();                             // the last column has been read
                s_o[wave][lane] = o;
                if (lane == 0) {
                    s_m[wave] = m;
                    s_l[wave] = ll;
                }
                __syncthreads();
                if (wave) continue;
                m = s_m[0];
#pragma unroll
                for (int w = 1; w < WAVES; ++w) m = fmaxf(m, s_m[w]);
                o = f2{0.f, 0.f};
                ll = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) {
                    const float f = __builtin_amdgcn_exp2f(s_m[w] - m);
                    o += s_o[w][lane] * f;
                    ll += s_l[w] * f;
                }
            }
            const int r = col / G, hh = col - r * G;
            *reinterpret_cast<f2*>(a.o + ((int64_t)(row0 + r) * NH + kvh * G + hh) * HD + 2 * lane) = o * (1.0f / ll);
        }
        done += all;
    }
}

// ---- host side ----

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int kFewCols = 64;                   // columns per session up to which a session's waves share them
constexpr int kAimWgs = 512;                   // workgroups aimed at: two per CU
constexpr int kMinShare = 4;                   // tiles: one per wave
constexpr int kJoinWgs = 2048;                 // a launch full of the chip
constexpr int kWideBlocks = 2;                 // 16-column blocks per wave of the wide form

// What a call of these counts runs with: the columns of a workgroup and the
// workgroups per kv head.
struct Shape {
    int blocks, cols, slots;
    bool wide;
};
Shape shape(int n_sess, int n_rows, int max_q) {
    Shape f{};
    const int64_t cols = (int64_t)max_q * G;
    f.wide = cols > kFewCols;
    f.blocks = f.wide ? kWideBlocks : cols <= 16 ? 1 : cols <= 32 ? 2 : 4;
    f.cols = 16 * f.blocks * (f.wide ? WAVES : 1);
    const int64_t groups = f.wide ? (int64_t)n_rows * G / f.cols + n_sess : n_sess;
    f.slots = (int)(kAimWgs / NKV + groups);
    return f;
}

struct Layout {
    size_t info, ml, acc, total;
};
Layout layout(const Shape& f, int n_sess) {
    Layout w{};
    const size_t rows = (size_t)NKV * f.slots * f.cols;
    w.ml = ((size_t)n_sess * sizeof(i4) + 255) / 256 * 256;
    w.acc = w.ml + (rows * sizeof(f2) + 255) / 256 * 256;
    w.total = w.acc + rows * HD * sizeof(float);
    return w;
}

Q8Args attn_args(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* n_keys,
                 int n_sess, int layer, int nb, float* o) {
    NOVA_REQUIRE(q && pool && tables && n_keys && o);
    NOVA_REQUIRE(aligned16(q) && aligned16(pool) && aligned16(o));
    NOVA_REQUIRE(layer >= 0 && layer < Model::L && nb > 0 && table_stride > 0 && table_stride <= (1 << 27));
    NOVA_REQUIRE((int64_t)n_sess * table_stride <= (int64_t)1 << 32);
    Q8Args a{};
    a.q = q;
    a.pool = pool + (int64_t)layer * nb * kQ8Page;
    a.tables = tables;
    a.table_stride = table_stride;
    a.n_keys = n_keys;
    a.n_sess = n_sess;
    a.nb = nb;
    a.o = o;
    a.gw = kAimWgs / NKV;
    a.min_share = kMinShare;
    return a;
}

template <bool kCausal>
void launch(Q8Args a, void* workspace, hipStream_t s) {
    const Shape f = shape(a.n_sess, a.rows.n_rows, a.max_q);
    const Layout w = layout(f, a.n_sess);
    char* ws = static_cast<char*>(workspace);
    a.slots = f.slots;
    a.info = reinterpret_cast<i4*>(ws + w.info);
    a.ml = reinterpret_cast<f2*>(ws + w.ml);
    a.acc = reinterpret_cast<float*>(ws + w.acc);
    const dim3 grid(NKV, f.slots);
    if constexpr (kCausal) {
        if (f.wide) hipLaunchKernelGGL((q8_attn_kernel<kWideBlocks, true, true>), grid, dim3(THREADS), 0, s, a);
        else if (f.blocks == 4) hipLaunchKernelGGL((q8_attn_kernel<4, true, false>), grid, dim3(THREADS), 0, s, a);
        else if (f.blocks == 2) hipLaunchKernelGGL((q8_attn_kernel<2, true, false>), grid, dim3(THREADS), 0, s, a);
    }
    if (f.blocks == 1) hipLaunchKernelGGL((q8_attn_kernel<1, kCausal, false>), grid, dim3(THREADS), 0, s, a);
    NOVA_LAUNCHED();
    const int64_t columns = (int64_t)a.rows.n_rows * NH;
    const unsigned join = (unsigned)std::min<int64_t>(f.wide ? (columns + WAVES - 1) / WAVES : columns, kJoinWgs);
    if (f.wide) hipLaunchKernelGGL(q8_join_kernel<true>, dim3(join), dim3(THREADS), 0, s, a, f.cols);
    else hipLaunchKernelGGL(q8_join_kernel<false>, dim3(join), dim3(THREADS), 0, s, a, f.cols);
    NOVA_LAUNCHED();
}

}  // namespace
}  // namespace nova

using namespace nova;

extern "C" {

size_t attn_decode_q8_workspace_bytes(int n_sess) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535);
    return layout(shape(n_sess, n_sess, 1), n_sess).total;
}

size_t attn_chunk_q8_workspace_bytes(int n_sess, int n_rows, int max_q) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && n_rows >= 0 && max_q >= 0 && max_q <= n_rows);
    return layout(shape(n_sess, n_rows, max_q), n_sess).total;
}

void launch_attn_decode_q8_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                 const int32_t* n_keys, int n_sess, int layer, int nb, float* o, void* workspace,
                                 nova_stream_t s) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535);
    Q8Args a = attn_args(q, pool, tables, table_stride, n_keys, n_sess, layer, nb, o);
    NOVA_REQUIRE(workspace && aligned16(workspace));
    a.rows = Q8Rows{nullptr, 1, n_sess};
    a.max_q = 1;
    launch<false>(a, workspace, reinterpret_cast<hipStream_t>(s));
}

void launch_attn_chunk_q8_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                const int32_t* n_past, const int32_t* row_off, int n_sess, int n_rows, int max_q,
                                int layer, int nb, float* o, void* workspace, nova_stream_t s) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && n_rows >= 0 && n_rows <= (1 << 24));
    NOVA_REQUIRE(max_q >= 0 && max_q <= n_rows);
    NOVA_REQUIRE(row_off || n_rows % n_sess == 0);
    Q8Args a = attn_args(q, pool, tables, table_stride, n_past, n_sess, layer, nb, o);
    NOVA_REQUIRE(workspace && aligned16(workspace));
    if (n_rows == 0 || max_q == 0) return;
    a.rows = Q8Rows{row_off, n_rows / n_sess, n_rows};
    a.max_q = max_q;
    launch<true>(a, workspace, reinterpret_cast<hipStream_t>(s));
}

}  // extern "C"
