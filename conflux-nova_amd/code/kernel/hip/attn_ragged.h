// attn_ragged.h -- what the attention kernels over quantised pages share, whatever the
// page format: the ragged batch, how its work is cut into workgroups, and the launches
// that join the pieces.
//
// Two kernels per format, by the columns (query rows x heads of a kv head) that a session
// may have.  "few": a workgroup's waves share its columns and split the keys; up to 32 columns, all in one
// workgroup (8-bit pages), or 16 to a workgroup and up to 64 over short tables (4-bit pages).  "many": 64
// columns a workgroup, all waves over the same keys.  A piece of a session's (or group's)
// work leaves {reference m, sum of 2^(s - m)} and the weighted sum of values per column in
// the workspace.
//
// Everything here has internal linkage: each format's source compiles its own, with its own
// kMinPiece (many columns: fewest tiles of a piece of a group) and kGroupTiles (what a group
// costs beside its tiles, in tiles), defined before this header.
#pragma once
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdint>
#include <type_traits>
#include <utility>

#include "check.h"
#include "kv_ragged.h"
#include "model.h"

namespace nova {
namespace {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int NH = Model::NH, NKV = Model::NKV, HD = Model::HD, G = Model::G;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int WAVES = 4;
constexpr int THREADS = 64 * WAVES;
constexpr int TILE = 64;                       // keys of a wave's step: four pages
constexpr int kTilePages = TILE / kKvBlock;
// Workgroups aimed at: two per CU (4-bit pages with four: 16 ragged sessions 21.6 us instead of 17.9, drafts 41.3,
// 32.3, short mixed prompts 49.6, 35.5, 8 x 512 rows 255, 238).  Of the 8-bit form with two blocks of columns
// one runs per CU, as it takes the registers of both, so its parts go through in two rounds.
constexpr int kAimWgs = 512;
constexpr int DB = HD / 16;                    // 16-dim blocks of the output
constexpr int kManyCols = 16 * WAVES;          // columns of a workgroup where there are many
constexpr float kUnset = -3.40282347e38f;      // reference of a column without keys, where states are joined: below every other
constexpr int kAccRow = HD + 4;                // floats per column in LDS: rows on different banks
static_assert(HD == 128 && kTilePages == 4 && G <= 16, "tile layout");

struct AttnArgs {
    const float* q;            // [n_rows][NH][HD]
    const uint8_t* pool;       // the layer's first page
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* n_keys;     // decode: keys of each session; chunk: its prefix
    RaggedRows rows;
    int max_q;
    int n_sess;
    int nb;
    int gw;                    // few columns: workgroups aimed at per kv head; many: workgroups per kv head
    int min_share;             // fewest tiles of a workgroup that shares a session
    int slots;                 // partial results per kv head
    float* o;
    i4* info;                  // few: [n_sess] {first slot, parts, rows, first row}; many: [2 gw] {session, group, its end, columns}
    f2* ml;                    // [NKV][slots][cols] {reference, sum}
    float* acc;                // [NKV][slots][cols][HD]
};

// ---- small cross-lane helpers ----

// the same of doubles, whole numbers here, by their halves
template <int kCtrl, int kRows>
__device__ __forceinline__ double dpp(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kCtrl, kRows, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), kCtrl, kRows, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double scan_incl(double v) {
    v += dpp<0x111, 0xf>(v);
    v += dpp<0x112, 0xf>(v);
    v += dpp<0x114, 0xf>(v);
    v += dpp<0x118, 0xf>(v);
    v += dpp<0x142, 0xa>(v);
    v += dpp<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ double read_lane(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
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

// over all lanes
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xf, 0xf, true)));   // row_ror 8, 4, 2, 1
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x124, 0xf, 0xf, true)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x122, 0xf, 0xf, true)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x121, 0xf, 0xf, true)));
    return rows_max(v);
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
__device__ __forceinline__ Session session_of(const AttnArgs& a, int i) {
    Session s;
    s.rows = min(row_count(a.rows, i), a.max_q);
    s.row0 = row_first(a.rows, i);
    const int n = min(max(a.n_keys[i], 0), 1 << 30);
    const int64_t most = a.table_stride * kKvBlock, all = (int64_t)n + (kCausal ? s.rows : 0);
    s.keys = (int)(all < most ? all : most);
    s.past = kCausal ? n : s.keys - 1;
    return s;
}

struct Part {
    int sess;                  // < 0: nothing to do
    int index, parts;          // part `index` of `parts` of the session's keys
    Session s;
};

// Few columns: the session and part of a slot.  With T tiles in the batch and gw
// workgroups aimed at, a session of t tiles is cut into ceil(t / share) parts,
// share = max(ceil(T / gw), min_share) or up to half more, so that no workgroup has more
// than that whatever the lengths, and at most gw + n_sess slots are used.  Every wave works it
// out for itself, 64 sessions at a time.
template <bool kCausal>
__device__ __forceinline__ Part find_part(const AttnArgs& a, int slot) {
    const int lane = threadIdx.x & 63;
    Session s{0, 0, 0, 0};
    int tiles = 0;
    auto load = [&](int base) {
        s = Session{0, 0, 0, 0};
        if (base + lane < a.n_sess) s = session_of<kCausal>(a, base + lane);
        tiles = s.rows > 0 ? (s.keys + TILE - 1) / TILE : 0;
    };
    int total = 0;
    for (int base = 0; base < a.n_sess; base += 64) {
        load(base);
        total += __builtin_amdgcn_readlane(scan_incl(tiles), 63);
    }
    // Whole tiles for each wave (nine tiles last as long as twelve), and no more parts
    // than workgroups that run at once, as one that has to wait may double the time, but
    // for that no more than half a share on top: where the sessions alone fill the chip,
    // parts of the first size that wait cost less than sessions that are not cut.
    const int least = (max((total + a.gw - 1) / a.gw, a.min_share) + WAVES - 1) / WAVES * WAVES;
    int share = least;
    auto parts_of = [&] { return s.rows > 0 ? max((tiles + share - 1) / share, 1) : 0; };
    if (a.n_sess <= 64) {
        const int step = max(least / 16 / WAVES, 1) * WAVES;
        while (__builtin_amdgcn_readlane(scan_incl(parts_of()), 63) > a.gw) {
            share += step;
            if (share > least + least / 2) {
                share = least;
                break;
            }
        }
    }
    int before = 0;
    for (int base = 0; base < a.n_sess; base += 64) {
        if (a.n_sess > 64) load(base);
        const int parts = parts_of();
        const int incl = before + scan_incl(parts);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(incl > slot);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            Part p;
            p.sess = base + l;
            p.parts = __builtin_amdgcn_readlane(parts, l);
            p.index = slot - (__builtin_amdgcn_readlane(incl, l) - p.parts);
            p.s.keys = __builtin_amdgcn_readlane(s.keys, l);
            p.s.past = __builtin_amdgcn_readlane(s.past, l);
            p.s.rows = __builtin_amdgcn_readlane(s.rows, l);
            p.s.row0 = __builtin_amdgcn_readlane(s.row0, l);
            return p;
        }
        before = __builtin_amdgcn_readlane(incl, 63);
    }
    return Part{-1, 0, 0, {0, 0, 0, 0}};
}

// Many columns: a session's columns in groups of C = kManyCols, group g over the keys up to its
// last row's.  The batch's work is one line, group after group, of which each
// workgroup gets the same length, so a group may be shared by workgroups that
// follow each other, and each of them has at most two groups in part.  The cost of
// group g is counted as G past + C (g + 1) (G times the keys its last row sees,
// where rows do not end inside a group) and as much as kGroupTiles tiles for its
// start and end, whose sums have a closed form; everything is in whole numbers, so
// that neighbours agree on where one stops and the other begins.
struct Place {
    int sess, group, tile;     // sess == n_sess: the end
};

__device__ __forceinline__ Place uniform(const Place& p) {
    return Place{__builtin_amdgcn_readfirstlane(p.sess), __builtin_amdgcn_readfirstlane(p.group),
                 __builtin_amdgcn_readfirstlane(p.tile)};
}

__device__ __forceinline__ int n_groups(const Session& s) {
    return (s.rows * G + kManyCols - 1) / kManyCols;
}
// tiles of group g
__device__ __forceinline__ int group_tiles(const Session& s, int g) {
    return (min(s.past + (min((g + 1) * kManyCols, s.rows * G) - 1) / G + 1, s.keys) + TILE - 1) / TILE;
}
// Cost of the first n groups, in a double: whole numbers below 2^53, exact.
__device__ __forceinline__ double flat_cost(const Session& s) { return (double)G * s.past + G * TILE * kGroupTiles; }
__device__ __forceinline__ double groups_cost(const Session& s, int n) {
    return (double)n * flat_cost(s) + 0.5 * kManyCols * ((double)n * (n + 1));
}

// where cost x of the line lies in session s, which begins at x = 0
__device__ __forceinline__ void place_in(const Session& s, double x, Place& p) {
    const double half = 0.5 * kManyCols, b = flat_cost(s) + half;
    int g = (int)((__builtin_sqrt(b * b + 4.0 * half * x) - b) / (2.0 * half));      // an estimate
    g = min(max(g, 0), n_groups(s) - 1);
    while (g > 0 && groups_cost(s, g) > x) --g;
    while (g + 1 < n_groups(s) && groups_cost(s, g + 1) <= x) ++g;
    const double lo = groups_cost(s, g), cost = groups_cost(s, g + 1) - lo;
    const int tiles = group_tiles(s, g);
    // no piece of fewer than kMinPiece tiles: it would cost more than it evens out
    int t = min((int)(((x - lo) * tiles) / cost), tiles);
    t = t < kMinPiece ? 0 : tiles - t < kMinPiece ? tiles : t;
    p.group = g;
    p.tile = t;
}

// The stretch of workgroup w: from `from` to before `to`.  The grid's gw workgroups
// are all used where each gets min_share tiles or more.
__device__ __forceinline__ void find_stretch(const AttnArgs& a, int w, Place& from, Place& to) {
    const int lane = threadIdx.x & 63;
    Session s{0, 0, 0, 0};
    double incl = 0;
    auto load = [&](int base) {                              // costs up to and with the lane's session
        s = Session{0, 0, 0, 0};
        if (base + lane < a.n_sess) s = session_of<true>(a, base + lane);
        incl = scan_incl(groups_cost(s, n_groups(s)));
    };
    double total = 0;
    for (int base = 0; base < a.n_sess; base += 64) {
        load(base);
        total += read_lane(incl, 63);
    }
    const int use = (int)fmin((double)a.gw, fmax(total / ((double)(G * TILE) * a.min_share), 1.0));
    from = to = Place{a.n_sess, 0, 0};
    if (w >= use) return;
    // whole numbers, the same for the workgroup that stops here and the one that starts
    const double x0 = __builtin_floor((total * w) / use), x1 = __builtin_floor((total * (w + 1)) / use);
    double before = 0;
    for (int base = 0; base < a.n_sess; base += 64) {
        if (a.n_sess > 64) load(base);
        auto find = [&](double x, Place& p) {
            x -= before;
            const uint64_t hit = __builtin_amdgcn_ballot_w64(incl > x);
            if (x < 0 || !hit) return;
            const int l = __builtin_ctzll(hit);
            Session t;
            t.keys = __builtin_amdgcn_readlane(s.keys, l);
            t.past = __builtin_amdgcn_readlane(s.past, l);
            t.rows = __builtin_amdgcn_readlane(s.rows, l);
            t.row0 = 0;
            p.sess = base + l;
            place_in(t, x - (read_lane(incl, l) - groups_cost(t, n_groups(t))), p);
        };
        find(x0, from);
        find(x1, to);
        before += read_lane(incl, 63);
    }
    from = uniform(from);
    to = uniform(to);
}

// ---- table entries, pieces ----

// Table entries, 64 at a time in a register: page pg (per lane, not before the
// last call's) of the session.
struct Pages {
    const int32_t* table;
    int last, nb;              // the last page with a key; pages of the pool
    int win, held;
    __device__ __forceinline__ Pages(const AttnArgs& a, int sess, int keys)
        : table(a.tables + sess * a.table_stride), last((keys - 1) >> kKvBlockShift), nb(a.nb), win(-64), held(0) {}
    __device__ __forceinline__ void reach(int pg) {          // uniform: pages pg .. pg + 3 come next
        if (pg + kTilePages > win + 64) {
            win = pg;
            held = table[min(pg + (int)(threadIdx.x & 63), last)];
        }
    }
    // page of the pool; an entry outside it reads page 0
    __device__ __forceinline__ int operator[](int pg) const {
        const int v = __shfl(held, min(pg, last) - win, 64);
        return (unsigned)v < (unsigned)nb ? v : 0;
    }
};

// 2^d, d <= 0, for a state moved to a reference -d higher.  In halves where it may be
// below fp32 and leave something that counts: for sums of weights, which are 2^98 at
// most and may count at 2^-100, and for sums of products between waves, whose units differ.
struct Factor {
    float half;
    __device__ __forceinline__ explicit Factor(float d) : half(__builtin_amdgcn_exp2f(0.5f * d)) {}
    template <class T>
    __device__ __forceinline__ T operator*(T v) const { return v * half * half; }
};

// joins pieces {reference, sum of weights}, v into the state m, l, o
template <int N, class V>
__device__ __forceinline__ void join(float& m, float& l, V& o, const f2 (&x)[N], const V (&v)[N]) {
    float to = m;
#pragma unroll
    for (int k = 0; k < N; ++k) to = fmaxf(to, x[k][0]);
    const Factor f(m - to);
    l = f * l;
    o = f * o;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const Factor f(x[k][0] - to);
        l += f * x[k][1];
        o += f * v[k];
    }
    m = to;
}

template <bool kOnce>
__device__ __forceinline__ i4 page_load(const uint8_t* p) {
    if constexpr (kOnce) return __builtin_nontemporal_load(reinterpret_cast<const i4*>(p));
    else return *reinterpret_cast<const i4*>(p);
}

// Joins the parts of the sessions that were cut: a workgroup per column of all kv
// heads, its waves taking every fourth part.
__global__ void __launch_bounds__(THREADS) few_join_kernel(AttnArgs a, int cols) {
    __shared__ f2 s_o[WAVES][64];
    __shared__ float s_l[WAVES], s_m[WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    int64_t done = 0;                                        // columns of the sessions before this batch of 64
    for (int base = 0; base < a.n_sess; base += 64) {
        i4 in = i4{0, 0, 0, 0};
        if (base + lane < a.n_sess && row_count(a.rows, base + lane) > 0) in = a.info[base + lane];
        const int mine = in[1] > 1 ? in[2] * NH : 0;
        const int incl = scan_incl(mine);
        const int all = __builtin_amdgcn_readlane(incl, 63);
        int u = (int)((blockIdx.x + gridDim.x - done % gridDim.x) % gridDim.x);
        for (; u < all; u += gridDim.x) {                    // uniform over the workgroup
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(incl > u));
            const int e = u - (__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(mine, l));
            const int slot0 = __builtin_amdgcn_readlane(in[0], l), parts = __builtin_amdgcn_readlane(in[1], l);
            const int n_cols = __builtin_amdgcn_readlane(in[2], l) * G, row0 = __builtin_amdgcn_readlane(in[3], l);
            const int kvh = e / n_cols, col = e % n_cols;
            if (slot0 + parts > a.slots) continue;           // offsets that do not add up
            const int64_t from = ((int64_t)kvh * a.slots + slot0) * cols + col;
            float m = kUnset, ll = 0.f;
            f2 o = f2{0.f, 0.f};
            for (int p = wave; p < parts; p += 4 * WAVES) {  // four parts' loads at a time
                f2 x[4], v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] = f2{kUnset, 0.f};
                    v[k] = f2{0.f, 0.f};
                    if (p + k * WAVES < parts) {
                        const int64_t at = from + (int64_t)(p + k * WAVES) * cols;
                        x[k] = a.ml[at];
                        v[k] = *reinterpret_cast<const f2*>(a.acc + at * HD + 2 * lane);
                    }
                }
                join(m, ll, o, x, v);
            }
            __syncthreads();                                 // the last column has been read
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
                const Factor f(s_m[w] - m);
                o += f * s_o[w][lane];
                ll += f * s_l[w];
            }
            const int r = col / G, hh = col - r * G;
            *reinterpret_cast<f2*>(a.o + ((int64_t)(row0 + r) * NH + kvh * G + hh) * HD + 2 * lane) = o * (1.0f / ll);
        }
        done += all;
    }
}

// Joins the pieces of groups that several workgroups had: the one that began a
// group names it, the next ones follow until one has its end.  32 lanes per column,
// and up to eight teams of them share a column's pieces, as many as its pieces need
// and there are workgroups for.
// Which of the next 64 stretches have a piece is read at once, and a team's pieces
// eight at a time: the launch lasts as long as its memory latencies in a row, 2.5 us
// each (8 rows behind 30000 keys, 7B, 128 pieces a group: the call takes 59 us with one
// team, 28 with eight; without teams, 16 and 32 pieces at a time 56 and 58).
constexpr int kJoinRows = THREADS / (HD / 4);
static_assert(kJoinRows == 8, "columns or teams of a workgroup");
__global__ void __launch_bounds__(THREADS) many_join_kernel(AttnArgs a) {
    constexpr int COLS = kManyCols, kAtOnce = 8, kBatches = (kAimWgs / NKV + 63) / 64;
    __shared__ f4 s_o[kJoinRows][HD / 4];
    __shared__ f2 s_ml[kJoinRows];
    const int lane = threadIdx.x & 63, row = threadIdx.x / (HD / 4), d = threadIdx.x % (HD / 4);
    i4 begun[kBatches];                                      // the groups that stretch 64 b + lane leaves open
#pragma unroll
    for (int b = 0; b < kBatches; ++b) {
        begun[b] = i4{-1, 0, 0, 0};
        if (64 * b + lane < a.gw) begun[b] = a.info[2 * (64 * b + lane) + 1];
    }
    // Columns of a workgroup: 8, or fewer for a group of more than 8 pieces, so that a
    // team has up to 8 (as many stretches lie before the next open group at most).
    int log[kBatches], later = a.gw;
#pragma unroll
    for (int b = kBatches - 1; b >= 0; --b) {
        const uint64_t open = __builtin_amdgcn_ballot_w64(begun[b][0] >= 0), behind = open >> lane >> 1;
        const int run = behind ? __builtin_ctzll(behind) + 1 : later - (64 * b + lane);
        log[b] = run <= 8 ? 3 : run <= 16 ? 2 : run <= 32 ? 1 : 0;
        if (open) later = 64 * b + __builtin_ctzll(open);
    }
    // a workgroup's units, up to and with stretch 64 b + lane's; no more than workgroups
    int incl[kBatches], units = 0;
    auto count = [&](int more) {
        units = 0;
#pragma unroll
        for (int b = 0; b < kBatches; ++b) {
            log[b] = min(log[b] + more, 3);
            incl[b] = units + scan_incl(begun[b][0] >= 0 ? ((begun[b][3] + (1 << log[b]) - 1) >> log[b]) * NKV : 0);
            units = __builtin_amdgcn_readlane(incl[b], 63);
        }
    };
    count(0);
    for (int i = 0; i < 3 && units > (int)gridDim.x; ++i) count(1);
    for (int u = blockIdx.x; u < units; u += gridDim.x) {    // uniform over the workgroup
        int w = -1, e = 0, sess = 0, group = 0, cols = 0, wide_log = 3;
#pragma unroll
        for (int b = 0; b < kBatches; ++b) {
            const uint64_t hit = __builtin_amdgcn_ballot_w64(incl[b] > u);
            if (w >= 0 || !hit) continue;
            const int l = __builtin_ctzll(hit);
            w = 64 * b + l;
            sess = __builtin_amdgcn_readlane(begun[b][0], l);
            group = __builtin_amdgcn_readlane(begun[b][1], l);
            cols = __builtin_amdgcn_readlane(begun[b][3], l);
            wide_log = __builtin_amdgcn_readlane(log[b], l);
            e = u - (__builtin_amdgcn_readlane(incl[b], l) - ((cols + (1 << wide_log) - 1) >> wide_log) * NKV);
        }
        const int wide = 1 << wide_log, teams = kJoinRows >> wide_log, team = row & (teams - 1);
        const int per = (cols + wide - 1) >> wide_log, kvh = e / per, cc = min(e % per * wide + (row >> __builtin_ctz(teams)), COLS - 1);
        const int64_t at = (int64_t)kvh * a.slots * COLS + cc;
        const Session s = session_of<true>(a, sess);
        float m = kUnset, l = 0.f;
        f4 o = f4{0.f, 0.f, 0.f, 0.f};
        if (team == 0 && cc < cols) {
            const int64_t from = at + (int64_t)(2 * w + 1) * COLS;
            const f2 x = a.ml[from];
            o = *reinterpret_cast<const f4*>(a.acc + from * HD + 4 * d);
            m = x[0];
            l = x[1];
        }
        for (int base = w + 1; base < a.gw; base += 64) {
            i4 next = i4{-1, 0, 0, 0};
            if (base + lane < a.gw) next = a.info[2 * (base + lane)];
            const bool ours = next[0] == sess && next[1] == group;           // others: too short to have a tile of it
            const uint64_t all = __builtin_amdgcn_ballot_w64(ours);
            const int rank = __builtin_popcountll(all & (((uint64_t)1 << lane) - 1));
            uint64_t todo = 0;                               // this team's
            for (int t = 0; t < teams; ++t) {
                const uint64_t x = __builtin_amdgcn_ballot_w64(ours && (rank & (teams - 1)) == t);
                if (t == team) todo = x;
            }
            if (cc >= cols) todo = 0;
            while (__builtin_amdgcn_ballot_w64(todo != 0)) {
                f2 x[kAtOnce];
                f4 p[kAtOnce];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    x[k] = f2{kUnset, 0.f};
                    p[k] = f4{0.f, 0.f, 0.f, 0.f};
                    if (todo) {
                        const int64_t from = at + (int64_t)(2 * (base + __builtin_ctzll(todo))) * COLS;
                        x[k] = a.ml[from];
                        p[k] = *reinterpret_cast<const f4*>(a.acc + from * HD + 4 * d);
                        todo &= todo - 1;
                    }
                }
                join(m, l, o, x, p);
            }
            if (__builtin_amdgcn_ballot_w64(ours && next[2])) break;         // the group's end
        }
        if (teams > 1) {
            __syncthreads();                                 // the last unit has been read
            s_o[row][d] = o;
            if (d == 0) s_ml[row] = f2{m, l};
            __syncthreads();
            if (team) continue;
            for (int t = 1; t < teams; ++t) {
                const f2 x[1] = {s_ml[row + t]};
                const f4 p[1] = {s_o[row + t][d]};
                join(m, l, o, x, p);
            }
        }
        const int col = group * COLS + cc;
        if (cc >= cols || col >= s.rows * G) continue;
        const int r = col / G, hh = col - r * G;
        *reinterpret_cast<f4*>(a.o + ((int64_t)(s.row0 + r) * NH + kvh * G + hh) * HD + 4 * d) = o * (1.0f / l);
    }
}

// ---- host side ----

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Columns per session up to which a workgroup's waves share them.  At 17 to 32 columns
// the other kernel is faster behind many long sessions (9 x 4400 keys, 4 rows, 7B: 29.5
// instead of 34.2 us; 24 x 3000: 38.1, 44.5) and slower for few or short ones (1 x 30000: 57.3,
// 37.3; 16 x 600: 19.8, 17.5; 32 x 100: 14.0, 11.5); the host knows the columns, not the keys.
constexpr int kFewCols = 32;
// Tiles of a workgroup that shares a session: one per wave.  Many columns, 12 prompts
// of up to 300 tokens (1.5B), 8-bit pages: 2 42.9 us, 4 43.1, 6 44.3, 8 57.4; 4-bit: 2 and 4 35.5.
constexpr int kMinShare = 4;
// A joining launch that fills the chip (4096: 16 sessions of 1 to 8 rows, 7B, 34.8 us instead
// of 34.4; 12 prompts of up to 300 tokens, 1.5B, 38.5, 37.4).
constexpr int kJoinWgs = 2048;

// What a call of these counts runs with: the columns of a workgroup and the partial
// results per kv head.
struct Shape {
    bool many;
    int cols, slots;
};
Shape shape(int n_sess, int max_q) {
    Shape f{};
    const int64_t cols = (int64_t)max_q * G;
    f.many = cols > kFewCols;
    f.cols = f.many ? kManyCols : cols <= 16 ? 16 : 32;
    f.slots = f.many ? 2 * (kAimWgs / NKV) : kAimWgs / NKV + n_sess;
    return f;
}

struct Layout {
    size_t info, ml, acc, total;
};
Layout layout(const Shape& f, int n_sess) {
    Layout w{};
    const size_t rows = (size_t)NKV * f.slots * f.cols;
    w.ml = ((size_t)(f.many ? f.slots : n_sess) * sizeof(i4) + 255) / 256 * 256;
    w.acc = w.ml + (rows * sizeof(f2) + 255) / 256 * 256;
    w.total = w.acc + rows * HD * sizeof(float);
    return w;
}

// page: bytes of a page of one layer
AttnArgs attn_args(int64_t page, const float* q, const uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* n_keys,
                 int n_sess, int layer, int nb, float* o) {
    NOVA_REQUIRE(q && pool && tables && n_keys && o);
    NOVA_REQUIRE(aligned16(q) && aligned16(pool) && aligned16(o));
    NOVA_REQUIRE(layer >= 0 && layer < Model::L && nb > 0 && table_stride > 0 && table_stride <= (1 << 27));
    NOVA_REQUIRE((int64_t)n_sess * table_stride <= (int64_t)1 << 32);
    AttnArgs a{};
    a.q = q;
    a.pool = pool + (int64_t)layer * nb * page;
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

}  // namespace
}  // namespace nova
