// kv_plan.hip -- a step's bookkeeping on the GPU: from the lengths of the sessions to
// pages given back and handed out, block tables, row offsets, positions and cache slots.
//
// Session i holds have tokens, keeps the first `keep` of them and adds `new`.  With
// pages(n) = ceil(n / 16) it gives back its pages [pages(keep), pages(have)) and takes
// pages(keep + new) - pages(keep).  The pages that are free are a stack; those given back go
// on top of it, in (session, page) order with the first on top, and pages are taken from the
// top in the same order, so a step that adds what the one before gave back gets the
// same pages.  Everything is prefix sums over the sessions, so there are no atomics and
// the result is the same every time.
//
// A workgroup does the sums (two passes over the sessions: what comes back, then what fits)
// and, for a small step, all the rest, out of registers and LDS.  Larger ones take two launches over
// the chip, as the stack must be whole before pages are taken from it: in the first, workgroups
// that sum for themselves what comes back put it on the stack, and one works out what fits;
// the second hands out pages and places rows.  It moves a few KB (16 sessions of a token each) to a
// MB, so latency bounds all of it: 3.6 us for those 16, 8.0 for 700 sessions and 60000 rows (3.8 and
// 4.2), where a launch that does nothing takes 2.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdint>

#include "check.h"
#include "model.h"
#include "nova_kernel.h"

namespace nova {
namespace {

typedef int i4 __attribute__((ext_vector_type(4)));

constexpr int PT = 1024;                       // threads of the workgroup that sums
constexpr int kPlanWaves = PT / 64;
constexpr uint32_t kNoneFits = ~0u;
static_assert(kPlanWaves == 16, "a wave's sums in a row of 16 lanes");
constexpr int FT = 256;                        // threads of the others
constexpr int kBackWgs = 64;                   // workgroups that give pages back, PT / kBackWgs sessions of every PT each
constexpr int kMine = PT / kBackWgs;
constexpr int kMostPasses = 64;                // PT sessions at a time
static_assert(kMostPasses * PT > 65535, "every session");
constexpr int kOffsets = 4096;                 // sessions whose row offsets fit a workgroup's LDS
// One launch up to this many rows and sessions.  One launch against two (us, one after another in a
// graph, 31 pages held; a launch more costs the host another 3): 16 sessions of 1 row 3.7, 5.2; of 64 4.6, 5.9;
// 64 of 16 6.3, 6.0; 256 of 4 5.7, 6.5; past it 64 of 32 7.1, 6.0, 256 of 8 6.6, 6.3, of 16 15.6, 6.5, 1000 of 1 10.4, 7.9.
constexpr int kSmallRows = 1024, kSmallSessions = 256;

struct PlanArgs {
    int32_t* tables;
    int64_t stride;
    const int32_t *have, *keep, *add;          // keep: or null
    int n_sess, max_rows, nb;
    int32_t* free_pages;
    const int32_t* n_free;
    int32_t *past, *keys, *row_off, *pos;
    int64_t* slots;
    int32_t* free_left;
    // workspace, between the two launches of a larger step
    i4* info;                                  // [n_sess] {first, held, pages back before, pages taken before}
    int32_t *ws_past, *ws_keys, *ws_off;       // what past, keys and row_off become (have may be one of them)
    int64_t* stack;                            // {free pages with those back, free pages left}
};

__device__ __forceinline__ int64_t pages_of(int64_t tokens) { return (tokens + kKvBlock - 1) >> kKvBlockShift; }

struct Wish {
    int64_t have, keep, add;
};
__device__ __forceinline__ Wish wish(const PlanArgs& a, int i) {
    const int64_t most = a.stride * kKvBlock;
    Wish w;
    w.have = min(max((int64_t)a.have[i], (int64_t)0), most);
    w.keep = a.keep ? min(max((int64_t)a.keep[i], (int64_t)0), w.have) : w.have;
    w.add = max((int64_t)a.add[i], (int64_t)0);
    if (w.keep + w.add > most) w.add = 0;                    // more than its table holds: nothing
    return w;
}

// Inclusive sums over the workgroup, in thread order; `total` for all threads.  They stop at
// 2^32 - 1, past every number of rows or pages that there is room for.
struct Pair {
    uint32_t a, b;
};
template <int kCtrl, int kRows = 0xf>
__device__ __forceinline__ void scan_step(uint32_t& v) {
    v = __builtin_elementwise_add_sat(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xf, false));
}
__device__ __forceinline__ uint32_t scan16(uint32_t v) {     // over each 16 lanes
    scan_step<0x111>(v);                                     // row_shr 1, 2, 4, 8
    scan_step<0x112>(v);
    scan_step<0x114>(v);
    scan_step<0x118>(v);
    return v;
}
__device__ __forceinline__ uint32_t scan64(uint32_t v) {
    v = scan16(v);
    scan_step<0x142, 0xa>(v);                                // row 0 -> 1, 2 -> 3
    scan_step<0x143, 0xc>(v);                                // rows 0, 1 -> 2, 3
    return v;
}
__device__ __forceinline__ Pair block_scan(Pair v, Pair* s_wave, Pair& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v.a = scan64(v.a);
    v.b = scan64(v.b);
    if (lane == 63) s_wave[wave] = v;
    __syncthreads();
    const Pair p = s_wave[lane & (kPlanWaves - 1)];
    const uint32_t a = scan16(p.a), b = scan16(p.b);
    total = Pair{(uint32_t)__builtin_amdgcn_readlane(a, kPlanWaves - 1), (uint32_t)__builtin_amdgcn_readlane(b, kPlanWaves - 1)};
    if (wave > 0) {                                          // uniform
        const int up = __builtin_amdgcn_readfirstlane(wave) - 1;
        v.a = __builtin_elementwise_add_sat(v.a, (uint32_t)__builtin_amdgcn_readlane(a, up));
        v.b = __builtin_elementwise_add_sat(v.b, (uint32_t)__builtin_amdgcn_readlane(b, up));
    }
    return v;
}

// the pages that session i gives back, onto the stack; one wave
__device__ __forceinline__ void give_back(const PlanArgs& a, int i, const i4& in, int64_t avail, int64_t n_free) {
    for (int p = in[0] + (int)(threadIdx.x & 63); p < in[1]; p += 64) {
        const int64_t at = avail - 1 - ((int64_t)in[2] + p - in[0]);
        if (at >= n_free) a.free_pages[at] = a.tables[i * a.stride + p];
    }
}
// the page that session i's nth new page is
__device__ __forceinline__ int taken(const PlanArgs& a, const i4& in, int64_t nth, int64_t avail) {
    return a.free_pages[avail - 1 - ((int64_t)in[3] + nth)];
}
__device__ __forceinline__ void hand_out(const PlanArgs& a, const i4* info, const int32_t* keys, int from, int step, int64_t avail) {
    for (int i = from; i < a.n_sess; i += step) {
        const i4 in = info[i];
        const int last = (int)pages_of(keys[i]);
        for (int p = in[0] + (int)(threadIdx.x & 63); p < last; p += 64) a.tables[i * a.stride + p] = taken(a, in, p - in[0], avail);
    }
}
// position and slot of row r; off: the rows' offsets
__device__ __forceinline__ void place_row(const PlanArgs& a, const i4* info, const int32_t* past, const int32_t* off, int r,
                                          int64_t avail) {
    int pos = -1;
    int64_t slot = -1;
    if (r < off[a.n_sess]) {
        int lo = 0, hi = a.n_sess - 1;                       // the last session that starts at r or before and has rows
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (off[mid] <= r) lo = mid;
            else hi = mid - 1;
        }
        pos = past[lo] + r - off[lo];
        const int p = pos >> kKvBlockShift;
        const i4 in = info[lo];
        const int page = p < in[0] ? a.tables[lo * a.stride + p] : taken(a, in, p - in[0], avail);
        if ((unsigned)page < (unsigned)a.nb) slot = (int64_t)page * kKvBlock + (pos & kKvBlockMask);
    }
    a.pos[r] = pos;
    a.slots[r] = slot;
}

// kAll: everything, for up to kSmallSessions sessions, whose numbers stay in registers and LDS.
// Else workgroup 0 leaves in the workspace what the second launch needs, and the others give pages back.
template <bool kAll>
__global__ void __launch_bounds__(PT) plan_kernel(PlanArgs a) {
    constexpr int kKept = kAll ? kSmallSessions : kMine * kMostPasses;
    __shared__ Pair s_wave[3][kPlanWaves];
    __shared__ int32_t s_off[kAll ? kKept + 1 : 1], s_past[kAll ? kKept : 1], s_keys[kAll ? kKept : 1];
    __shared__ __attribute__((aligned(16))) i4 s_info[kKept];
    const int tid = threadIdx.x;
    const int64_t n_free = min(max((int64_t)*a.n_free, (int64_t)0), (int64_t)a.nb);
    // what comes back
    int64_t back = 0;
    Wish w{0, 0, 0};
    i4 in = i4{0, 0, 0, 0};
    for (int base = 0; base < a.n_sess; base += PT) {
        const int i = base + tid;
        in = i4{0, 0, 0, 0};
        if (i < a.n_sess) {
            w = wish(a, i);
            in[0] = (int)pages_of(w.keep);
            in[1] = (int)pages_of(w.have);
        }
        Pair total;
        const int of = base / PT & 1;                        // (the last call's sums may still be read)
        const Pair sum = block_scan(Pair{(uint32_t)(in[1] - in[0]), 0}, s_wave[of], total);
        // (more than the stack holds is nowhere)
        in[2] = (int)min(back + sum.a - (in[1] - in[0]), (int64_t)a.nb);
        if (!kAll) {
            if (blockIdx.x == 0) {
                if (i < a.n_sess) a.info[i] = in;
            } else if (tid / kMine == (int)blockIdx.x - 1) s_info[base / PT * kMine + tid % kMine] = in;
        }
        back += total.a;
    }
    const int64_t avail = min(n_free + back, (int64_t)a.nb);
    if (!kAll && blockIdx.x > 0) {
        __syncthreads();
        const int kept = (a.n_sess + PT - 1) / PT * kMine;
        for (int j = tid >> 6; j < kept; j += kPlanWaves)     // (sessions behind the last hold nothing)
            give_back(a, j / kMine * PT + ((int)blockIdx.x - 1) * kMine + j % kMine, s_info[j], avail, n_free);
        return;
    }
    // What fits: the sessions before the first with which the sums of what was wished for pass the room, so
    // the sums up to a session that fits are those of what was granted.
    int64_t rows_before = 0, pages_before = 0;               // wished for by the sessions of the passes before
    Pair given{0, 0};                                        // rows, pages
    if (!kAll) __syncthreads();                              // s_wave is used again
    for (int base = 0; base < a.n_sess; base += PT) {
        const int i = base + tid;
        const bool real = i < a.n_sess;
        if (!kAll) w = real ? wish(a, i) : Wish{0, 0, 0};
        const int64_t rows = min(w.add, (int64_t)a.max_rows + 1);            // one too many is as good as more
        const int64_t more = pages_of(w.keep + rows) - pages_of(w.keep);
        Pair total;
        const Pair sum = block_scan(Pair{(uint32_t)rows, (uint32_t)more}, s_wave[kAll ? 1 : 0], total);
        const int64_t all_rows = rows_before + sum.a, all_pages = pages_before + sum.b;
        const bool fits = all_rows <= a.max_rows && all_pages <= avail;
        // what those that fit have together: with the wave's last of them, and the last wave's
        const uint64_t hits = __builtin_amdgcn_ballot_w64(fits);
        if (hits ? (tid & 63) == 63 - __builtin_clzll(hits) : (tid & 63) == 0)
            s_wave[2][tid >> 6] = hits ? Pair{(uint32_t)all_rows, (uint32_t)all_pages} : Pair{kNoneFits, 0};
        __syncthreads();
        const Pair fit = s_wave[2][tid & (kPlanWaves - 1)];
        const int fit_waves = __builtin_popcountll(__builtin_amdgcn_ballot_w64(fit.a != kNoneFits) & ((1u << kPlanWaves) - 1));
        if (fit_waves > 0)
            given = Pair{(uint32_t)__builtin_amdgcn_readlane(fit.a, fit_waves - 1),
                         (uint32_t)__builtin_amdgcn_readlane(fit.b, fit_waves - 1)};
        if (real) {
            const int keys = (int)(w.keep + (fits ? rows : 0)), end = (int)(fits ? all_rows : given.a);
            const int first = fits ? (int)(all_pages - more) : 0;
            (kAll ? a.past : a.ws_past)[i] = (int)w.keep;
            (kAll ? a.keys : a.ws_keys)[i] = keys;
            (kAll ? a.row_off : a.ws_off)[i + 1] = end;
            if constexpr (kAll) {
                in[3] = first;
                s_info[i] = in;
                s_past[i] = (int)w.keep;
                s_keys[i] = keys;
                s_off[i + 1] = end;
            } else a.info[i][3] = first;
        }
        rows_before += total.a;
        pages_before += total.b;
    }
    if (tid == 0) {
        if constexpr (kAll) {
            a.row_off[0] = 0;
            s_off[0] = 0;
            *a.free_left = (int)(avail - given.b);
        } else {
            a.ws_off[0] = 0;
            a.stack[0] = avail;
            a.stack[1] = avail - given.b;
        }
    }
    if constexpr (kAll) {
        __syncthreads();
        if (back > 0) {                                      // uniform
            for (int i = tid >> 6; i < a.n_sess; i += kPlanWaves) give_back(a, i, s_info[i], avail, n_free);
            __syncthreads();
        }
        hand_out(a, s_info, s_keys, tid >> 6, PT / 64, avail);
        for (int r = tid; r < a.max_rows; r += PT) place_row(a, s_info, s_past, s_off, r, avail);
    }
}

// workgroups below row_wgs: rows; the others: tables and what the sessions have now
__global__ void __launch_bounds__(FT) plan_rows_kernel(PlanArgs a, int row_wgs) {
    __shared__ int32_t s_off[kOffsets + 1];
    const int64_t avail = a.stack[0];
    if ((int)blockIdx.x >= row_wgs) {
        const int wgs = (int)gridDim.x - row_wgs, w = (int)blockIdx.x - row_wgs;
        for (int i = w * FT + (int)threadIdx.x; i <= a.n_sess; i += wgs * FT) {
            a.row_off[i] = a.ws_off[i];
            if (i == a.n_sess) *a.free_left = (int)a.stack[1];
            else {
                a.past[i] = a.ws_past[i];
                a.keys[i] = a.ws_keys[i];
            }
        }
        hand_out(a, a.info, a.ws_keys, w * (FT / 64) + (int)(threadIdx.x >> 6), wgs * (FT / 64), avail);
        return;
    }
    const bool here = a.n_sess <= kOffsets;
    if (here)
        for (int i = threadIdx.x; i <= a.n_sess; i += FT) s_off[i] = a.ws_off[i];
    __syncthreads();
    for (int r = blockIdx.x * FT + threadIdx.x; r < a.max_rows; r += row_wgs * FT) place_row(a, a.info, a.ws_past, here ? s_off : a.ws_off, r, avail);
}

constexpr int kWgs = 1024;                     // of the larger launches

// workspace: the stack's two numbers, then the sessions'
size_t info_at() { return 256; }
size_t past_at(int n_sess) { return info_at() + (size_t)n_sess * sizeof(i4); }
size_t bytes(int n_sess) { return past_at(n_sess) + (3 * (size_t)n_sess + 1) * sizeof(int32_t); }

}  // namespace
}  // namespace nova

using namespace nova;

extern "C" {

size_t kv_step_plan_workspace_bytes(int n_sess) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535);
    return bytes(n_sess);
}

void launch_kv_step_plan(int32_t* tables, int table_stride, const int32_t* n_have, const int32_t* n_keep,
                         const int32_t* n_new, int n_sess, int max_rows, int32_t* free_pages, const int32_t* n_free, int nb,
                         int32_t* n_past, int32_t* n_keys, int32_t* row_off, int32_t* pos, int64_t* slots,
                         int32_t* n_free_left, void* workspace, nova_stream_t s) {
    NOVA_REQUIRE(tables && n_have && n_new && free_pages && n_free && n_past && n_keys && row_off && n_free_left);
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && table_stride > 0 && table_stride <= (1 << 26));
    NOVA_REQUIRE((int64_t)n_sess * table_stride <= (int64_t)1 << 32);
    NOVA_REQUIRE(max_rows >= 0 && max_rows <= (1 << 24) && nb > 0 && nb <= (1 << 27));
    NOVA_REQUIRE((pos && slots) || max_rows == 0);
    NOVA_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0);
    char* ws = static_cast<char*>(workspace);
    int32_t* ws_past = reinterpret_cast<int32_t*>(ws + past_at(n_sess));
    const PlanArgs a{tables,  table_stride, n_have, n_keep,  n_new, n_sess, max_rows,    nb,
                     free_pages, n_free,       n_past, n_keys, row_off, pos,   slots,  n_free_left,
                     reinterpret_cast<i4*>(ws + info_at()), ws_past, ws_past + n_sess, ws_past + 2 * n_sess,
                     reinterpret_cast<int64_t*>(ws)};
    const hipStream_t st = reinterpret_cast<hipStream_t>(s);
    if (max_rows <= kSmallRows && n_sess <= kSmallSessions) {
        hipLaunchKernelGGL(plan_kernel<true>, dim3(1), dim3(PT), 0, st, a);
        NOVA_LAUNCHED();
        return;
    }
    hipLaunchKernelGGL(plan_kernel<false>, dim3(1 + kBackWgs), dim3(PT), 0, st, a);
    NOVA_LAUNCHED();
    const int sess_wgs = std::min((n_sess + FT / 64 - 1) / (FT / 64), kWgs);
    const int row_wgs = std::min((max_rows + FT - 1) / FT, kWgs);
    hipLaunchKernelGGL(plan_rows_kernel, dim3(row_wgs + sess_wgs), dim3(FT), 0, st, a, row_wgs);
    NOVA_LAUNCHED();
}

}  // extern "C"
