// kv_rows.h -- what the row kernels (append, read back) and the page kernels (copy on
// write, clear) over quantised pages share, whatever the page format.  Internal linkage:
// each format's source compiles its own.
#pragma once
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cstdint>
#include <memory>
#include <new>

#include "check.h"
#include "kv_ragged.h"
#include "model.h"
#include "nova_kernel.h"

namespace nova {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct RowArgs {
    uint8_t* pool;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* pos0;       // device [n_sess]: position of each session's first row
    RaggedRows rows;
    int n_sess;
    int layer;
    int nb;
    float* q;                  // RoPE: [n_rows][NH][HD], written rotated
    const float* k;            // store: [n_rows][NKV][HD]
    const float* v;
    const float* cs;           // RoPE: table rows [pos][HD/2]
    const float* sn;
    float* k_out;              // read back: [n_rows][NKV][HD]
    float* v_out;
};

// The page that workgroup `index` serves: the call's pages, session by session.
// A session with n rows from pos0 touches (pos0 + n - 1) / 16 - pos0 / 16 + 1
// pages.  Every wave scans the sessions 64 at a time, so the answer is
// wave-uniform; `sess` < 0 past the last page.
struct PageItem {
    int sess, page;            // session, logical page
    int pos0, row0, n;         // the session's first position, first row, rows
};
__device__ __forceinline__ PageItem page_item(const RowArgs& a, int index) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.n_sess; base += 64) {
        const int i = base + lane;
        int n = 0, p0 = 0, r0 = 0, pages = 0;
        if (i < a.n_sess) {
            p0 = a.pos0[i];
            r0 = row_first(a.rows, i);
            n = row_count(a.rows, i);
            // positions outside the session's table are left out
            if (p0 < 0) n = 0;
            const int64_t end = (int64_t)a.table_stride * kKvBlock;
            n = (int64_t)p0 + n > end ? (int)(end > p0 ? end - p0 : 0) : n;
            if (n > 0) pages = ((p0 + n - 1) >> kKvBlockShift) - (p0 >> kKvBlockShift) + 1;
        }
        const int incl = scan_incl(pages);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(before + incl > index);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            PageItem it;
            it.sess = base + l;
            it.pos0 = __builtin_amdgcn_readlane(p0, l);
            it.row0 = __builtin_amdgcn_readlane(r0, l);
            it.n = __builtin_amdgcn_readlane(n, l);
            it.page = (it.pos0 >> kKvBlockShift) + index - (before + __builtin_amdgcn_readlane(incl - pages, l));
            return it;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return PageItem{-1, 0, 0, 0, 0};
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Host checks and the grid of the row kernels.  A run of n rows touches at most
// (n + 30) / 16 pages.
RowArgs row_args(uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* pos0, const int32_t* row_off,
                 int n_sess, int n_rows, int layer, int nb) {
    NOVA_REQUIRE(pool && tables && pos0);
    NOVA_REQUIRE(aligned16(pool));
    NOVA_REQUIRE(layer >= 0 && layer < Model::L && nb > 0 && table_stride > 0 && table_stride <= (1 << 27));
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && n_rows >= 0 && n_rows <= (1 << 24));
    NOVA_REQUIRE(row_off || n_rows % n_sess == 0);
    RowArgs a{};
    a.pool = pool;
    a.tables = tables;
    a.table_stride = table_stride;
    a.pos0 = pos0;
    a.rows = RaggedRows{row_off, n_rows / n_sess, n_rows};
    a.n_sess = n_sess;
    a.layer = layer;
    a.nb = nb;
    return a;
}

unsigned page_bound(const RowArgs& a) {
    if (!a.rows.off) return (unsigned)((int64_t)a.n_sess * ((a.rows.uniform + 30) / 16));
    return (unsigned)(((int64_t)a.rows.n_rows + 30LL * std::min(a.n_sess, a.rows.n_rows)) / 16);
}

// ---- copy on write and clears of pages of kPage bytes a layer ----

constexpr int kOpsPerLaunch = 64;
struct CowOps {
    nova_cow_op op[kOpsPerLaunch];
};

// grid: x = chunks over a page's layers, y = op.  HBM-bound movement of 16 B per
// lane, as the fp16 pages are copied; block (0, y) patches the table entry.
template <int64_t kPage>
__global__ void __launch_bounds__(256)
cow_kernel(uint8_t* __restrict__ pool, int nb, int32_t* __restrict__ tables, CowOps ops) {
    const nova_cow_op o = ops.op[blockIdx.y];
    if (blockIdx.x == 0 && threadIdx.x == 0 && tables) tables[o.table_index] = o.dst;
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < Model::L * (kPage / 16);
         e += (int64_t)gridDim.x * blockDim.x) {
        const int64_t layer = e / (kPage / 16), off = e - layer * (kPage / 16);
        const u4 x = *reinterpret_cast<const u4*>(pool + (layer * nb + o.src) * kPage + 16 * off);
        *reinterpret_cast<u4*>(pool + (layer * nb + o.dst) * kPage + 16 * off) = x;
    }
}

template <int64_t kPage>
__global__ void __launch_bounds__(256)
zero_kernel(uint8_t* __restrict__ pool, int nb, const int32_t* __restrict__ pages) {
    const int pg = pages[blockIdx.y];
    if ((unsigned)pg >= (unsigned)nb) return;
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < Model::L * (kPage / 16);
         e += (int64_t)gridDim.x * blockDim.x) {
        const int64_t layer = e / (kPage / 16), off = e - layer * (kPage / 16);
        *reinterpret_cast<u4*>(pool + (layer * nb + pg) * kPage + 16 * off) = u4{0u, 0u, 0u, 0u};
    }
}

// workgroups per page over all layers: 8 vectors per thread
template <int64_t kPage>
constexpr int kCopyChunks = (int)((Model::L * (kPage / 16) + 256 * 8 - 1) / (256 * 8));

constexpr int kPagesPerLaunch = 65535;         // of clears: a launch's grid

template <int64_t kPage>
void cow_apply(uint8_t* pool, int nb, int32_t* tables_dev, const nova_cow_op* ops, int n_ops, hipStream_t s) {
    NOVA_REQUIRE(pool && aligned16(pool) && nb > 0 && n_ops >= 0);
    if (n_ops == 0) return;
    NOVA_REQUIRE(ops);
    // The copies of a call run side by side: a page written by one op may be
    // neither read nor written by another, nor be its own source.
    int32_t few[2 * kOpsPerLaunch];
    std::unique_ptr<int32_t[]> many(n_ops > kOpsPerLaunch ? new (std::nothrow) int32_t[2 * (size_t)n_ops] : nullptr);
    NOVA_REQUIRE(n_ops <= kOpsPerLaunch || many);
    int32_t* dst = many ? many.get() : few;
    int32_t* src = dst + n_ops;
    for (int e = 0; e < n_ops; ++e) {
        NOVA_REQUIRE(ops[e].src >= 0 && ops[e].src < nb);
        NOVA_REQUIRE(ops[e].dst >= 0 && ops[e].dst < nb);
        NOVA_REQUIRE(!tables_dev || ops[e].table_index >= 0);
        src[e] = ops[e].src;
        dst[e] = ops[e].dst;
    }
    std::sort(dst, dst + n_ops);
    std::sort(src, src + n_ops);
    for (int e = 0, f = 0; e < n_ops; ++e) {
        const bool dst_repeats = e > 0 && dst[e] == dst[e - 1];
        NOVA_REQUIRE(!dst_repeats);
        while (f < n_ops && src[f] < dst[e]) ++f;
        const bool dst_is_a_source = f < n_ops && src[f] == dst[e];
        NOVA_REQUIRE(!dst_is_a_source);
    }
    for (int base = 0; base < n_ops; base += kOpsPerLaunch) {
        const int n = n_ops - base < kOpsPerLaunch ? n_ops - base : kOpsPerLaunch;
        CowOps o{};
        std::copy(ops + base, ops + base + n, o.op);
        hipLaunchKernelGGL(cow_kernel<kPage>, dim3(kCopyChunks<kPage>, n), dim3(256), 0, s, pool, nb,
                           tables_dev, o);
        NOVA_LAUNCHED();
    }
}

template <int64_t kPage>
void zero_pages(uint8_t* pool, int nb, const int32_t* pages, int n_pages, hipStream_t s) {
    NOVA_REQUIRE(pool && aligned16(pool) && nb > 0 && n_pages >= 0);
    if (n_pages == 0) return;
    NOVA_REQUIRE(pages);
    for (int base = 0; base < n_pages; base += kPagesPerLaunch) {
        hipLaunchKernelGGL(zero_kernel<kPage>, dim3(kCopyChunks<kPage>, std::min(n_pages - base, kPagesPerLaunch)), dim3(256), 0,
                           s, pool, nb, pages + base);
        NOVA_LAUNCHED();
    }
}

}  // namespace
}  // namespace nova
