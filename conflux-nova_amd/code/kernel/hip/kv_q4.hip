// kv_q4.hip -- 4-bit pages (kv_q4.h): quantise K and V as they are written (alone or with
// RoPE), read rows back, copy-on-write page copies and page clears.
//
// Quantiser, per 32 values: a = max |x|, e the smallest integer with a <= 7 2^e, codes the
// values of the format nearest to x / 2^e, ties to the even code.  7 is the middle between 6 and
// the 8 that the format does not have, so that no value is off by more than half a step of
// its own size (with a <= 6 2^e, most blocks would spend an octave more on one value; with
// the exponent of a alone, values up to 8 2^e would be cut to 6).  e is held to 96; blocks whose
// e would be below -100 count as zeros.  x / 2^e is exact, and the rounding is the conversion
// instruction's.  A row that holds an infinity or a NaN gets the
// exponent byte 255 in all its blocks, so that it reads back as NaN and never as a
// finite value.
//
// Layout of the work: a workgroup takes one page of one session's call and one kv head, 16
// lanes per token; lane j holds dims 8j .. 8j + 7, four lanes a block.  K's codes leave as
// one word per lane; V's bytes hold two dims of one token each, 16 tokens together, so they
// go through LDS and leave as words where the call fills the page, byte by byte
// otherwise: no byte holds two tokens, so the page's other tokens stay as they are.
//
// What bounds it: HBM (4096 rows of 7B, rotation and append, 138 MB: 32 us, 4.3 TB/s, where a large
// copy reaches 5.1; one call after another, whose rows the caches still have, 25) or, for a step's few rows, a launch
// and three loads that wait for each other (16 rows 3.8 us).  The append alone: 4096 rows, 19 MB, 4.1 us from the
// caches, 16 rows 2.8.  The read back of 4096 rows, 19 MB, takes 7.5: twice what their bytes need; V comes out of
// LDS byte by byte, with bank conflicts (0.46 M).
#include <hip/hip_runtime.h>
#include <cstdint>
#include <type_traits>

#include "check.h"
#include "kv_q4.h"
#include "kv_rows.h"
#include "model.h"
#include "nova_kernel.h"
#include "rope_rows.h"

namespace nova {
namespace {

constexpr int NH = Model::NH, NKV = Model::NKV, HD = Model::HD;
constexpr int kLanes = 16;                     // lanes per token
constexpr int QT = kKvBlock * kLanes;          // threads of a workgroup
constexpr int kHeads = 4;                      // query heads of a workgroup
static_assert(QT == 256 && kLanes * 8 == HD, "one page per workgroup, 8 dims per lane");
static_assert(NH % kHeads == 0, "whole workgroups of query heads");

struct StoreArgs : RowArgs {
    const float* q_in;         // RoPE: [n_rows][NH][HD]
    int rot;
};

// 8 dims of a row as codes, dim 8j + e in bits 4e; byte: the exponent byte of the lane's block
__device__ __forceinline__ uint32_t quantise(const float (&x)[8], int& byte) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1, kLanes));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2, kLanes));
    uint32_t row = max(top, (uint32_t)__shfl_xor((int)top, 4, kLanes));
    row = max(row, (uint32_t)__shfl_xor((int)row, 8, kLanes));
    // exponent of a less 2, one more where its mantissa is above 1.75: a > 7 2^e
    byte = min((int)((top + 0x1fffffu) >> 23) - 2, kQ4MostExp);
    uint32_t w = 0;
    if (byte < kQ4LeastExp) byte = 0;
    else {
        const float unit = __uint_as_float((uint32_t)byte << 23);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], unit, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], unit, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], unit, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], unit, 3);
    }
    if (row >= 0x7f800000u) {
        byte = kQ4Nan;
        w = 0;
    }
    return w;
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const f4 a = *reinterpret_cast<const f4*>(p), b = *reinterpret_cast<const f4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = a[e];
        x[4 + e] = b[e];
    }
}

// V byte of dims 32 b + r and 32 b + 16 + r, from the token's 16 words of codes
__device__ __forceinline__ uint32_t v_byte(const uint32_t* token, int b, int r) {
    const int at = 4 * b + (r >> 3), sh = 4 * (r & 7);
    return ((token[at] >> sh) & 15u) | (((token[at + 2] >> sh) & 15u) << 4);
}

// Workgroups of a page: its kv heads, then (RoPE) kHeads query heads each, one after another in the
// grid, as their rows stand in memory.  Workgroups go round the 8 XCDs in turn, so a number
// of units that 8 divides would give each XCD the same units of every page, kv heads to some and
// query heads to others (7B, 4096 rows, one launch: 1, 2, 4, 8 heads: 44.1, 31.6, 32.1, 48.0 us, where 1
// and 8 are such numbers; 4 heads in an order of all pages of a head first: 33.4).
template <bool kRope>
constexpr int kUnits = NKV + (kRope ? NH / kHeads : 0);
static_assert(kUnits<true> % 8 != 0, "units spread over the XCDs");

// Workgroups of a call: its pages (an upper bound) times kUnits.  A launch has fewer than 2^32 threads, which the
// rotation and append of the 14B shape would pass from 13 million rows on (370 GB of them).
template <bool kRope>
unsigned store_wgs(const RowArgs& a) {
    const uint64_t wgs = (uint64_t)page_bound(a) * kUnits<kRope>;
    NOVA_REQUIRE(wgs * QT <= UINT32_MAX);
    return (unsigned)wgs;
}

// grid: store_wgs
template <bool kRope, RopeForm kForm>
__global__ void __launch_bounds__(QT) q4_store_kernel(StoreArgs a) {
    const PageItem it = page_item(a, blockIdx.x / kUnits<kRope>);
    if (it.sess < 0) return;
    const int head = blockIdx.x % kUnits<kRope>;
    const int t = threadIdx.x / kLanes, j = threadIdx.x % kLanes;
    const int pos = it.page * kKvBlock + t;
    const int first = max(it.pos0 - it.page * kKvBlock, 0);                   // tokens [first, last) of the page
    const int last = min(it.pos0 + it.n - it.page * kKvBlock, kKvBlock);
    const bool real = t >= first && t < last;
    const int64_t row = it.row0 + pos - it.pos0;
    if constexpr (kRope) {
        if (head >= NKV) {                                        // query heads
            if (!real) return;
            const int64_t at = (row * NH + (head - NKV) * kHeads) * HD, angle = row * (a.rot / 2);
            const int units = rope_units<kForm>(a.rot);
            for (int u = j; u < units; u += kLanes)
#pragma unroll
                for (int h = 0; h < kHeads; ++h)
                    rope_unit<kForm>(a.q_in + at + h * HD, a.q + at + h * HD, a.cs + angle, a.sn + angle, a.rot, u);
            return;
        }
    }
    float k[8] = {}, v[8] = {};                                              // the rows, requested beside the table entry
    if (real) {
        const int64_t at = (row * NKV + head) * HD;
        if constexpr (kRope) rope_dims8<kForm>(a.k + at, a.cs + row * (a.rot / 2), a.sn + row * (a.rot / 2), a.rot, j, k);
        else load8(a.k + at + 8 * j, k);
        load8(a.v + at + 8 * j, v);
    }
    const int phys = a.tables[it.sess * a.table_stride + it.page];
    if ((unsigned)phys >= (unsigned)a.nb) return;                            // no such page: nothing is written
    uint8_t* rec = a.pool + ((int64_t)a.layer * a.nb + phys) * kQ4Page + head * kQ4Rec;
    __shared__ uint32_t s_v[kKvBlock][kLanes];
    int ke, ve;
    const uint32_t kw = quantise(k, ke), vw = quantise(v, ve);
    s_v[t][j] = vw;
    if (real) {
        *reinterpret_cast<uint32_t*>(rec + t * 64 + 4 * j) = kw;
        if ((j & 3) == 0) {
            rec[kQ4KeOff + (t & 3) * 16 + (j >> 2) * 4 + (t >> 2)] = (uint8_t)ke;
            rec[kQ4VeOff + (j >> 2) * 16 + t] = (uint8_t)ve;
        }
    }
    __syncthreads();
    if (first == 0 && last == kKvBlock) {                                    // uniform over the workgroup
        const int b = threadIdx.x >> 6, r = (threadIdx.x >> 2) & 15, t0 = 4 * (threadIdx.x & 3);
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w |= v_byte(s_v[t0 + e], b, r) << (8 * e);
        *reinterpret_cast<uint32_t*>(rec + kQ4VOff + 4 * threadIdx.x) = w;
    } else if (real) {
#pragma unroll
        for (int b = 0; b < 4; ++b) rec[kQ4VOff + b * 256 + j * 16 + t] = (uint8_t)v_byte(s_v[t], b, j);
    }
}

// what a 4-bit code stands for, before its power of two
__device__ __forceinline__ float value(uint32_t code) {
    const uint32_t m = code & 7u;                            // m < 2: m / 2, else (1 or 1.5) 2^(m / 2 - 1)
    const float v = m < 2 ? 0.5f * (float)m : __uint_as_float(((126u + (m >> 1)) << 23) | ((m & 1u) << 22));
    return code & 8u ? -v : v;
}
__device__ __forceinline__ float power(uint32_t byte) {
    return byte == 0 ? 0.f : byte == (uint32_t)kQ4Nan ? __builtin_nanf("") : __uint_as_float(byte << 23);
}

// the reverse: every value is exact
__global__ void __launch_bounds__(QT) q4_load_kernel(RowArgs a) {
    const PageItem it = page_item(a, blockIdx.x);
    if (it.sess < 0) return;
    const int t = threadIdx.x / kLanes, j = threadIdx.x % kLanes;
    const int first = max(it.pos0 - it.page * kKvBlock, 0);
    const int last = min(it.pos0 + it.n - it.page * kKvBlock, kKvBlock);
    const int head = blockIdx.y;
    const int phys = page_or_0(a.tables + it.sess * a.table_stride, it.page, a.nb);
    const uint8_t* rec = a.pool + ((int64_t)a.layer * a.nb + phys) * kQ4Page + head * kQ4Rec;
    // every read of the record goes out before the first wait
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(rec + t * 64 + 4 * j);
    const uint32_t ke = rec[kQ4KeOff + (t & 3) * 16 + (j >> 2) * 4 + (t >> 2)], ve = rec[kQ4VeOff + (j >> 2) * 16 + t];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[kQ4KBytes];
    *reinterpret_cast<uint32_t*>(s_v + 4 * threadIdx.x) = *reinterpret_cast<const uint32_t*>(rec + kQ4VOff + 4 * threadIdx.x);
    __syncthreads();
    if (t < first || t >= last) return;
    const int64_t row = it.row0 + it.page * kKvBlock + t - it.pos0;
    f4 k[2], v[2];
    const float kp = power(ke), vp = power(ve);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        k[e / 4][e % 4] = value(kw >> (4 * e)) * kp;
        // dim 8j + e: of block j >> 2, bit 4 of it j >> 1
        const uint32_t b = s_v[(j >> 2) * 256 + (8 * (j & 1) + e) * 16 + t];
        v[e / 4][e % 4] = value(b >> (j & 2 ? 4 : 0)) * vp;
    }
    const int64_t at = (row * NKV + head) * HD + 8 * j;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        *reinterpret_cast<f4*>(a.k_out + at + 4 * e) = k[e];
        *reinterpret_cast<f4*>(a.v_out + at + 4 * e) = v[e];
    }
}

}  // namespace
}  // namespace nova

using namespace nova;

extern "C" {

size_t kv_q4_page_bytes(void) { return (size_t)kQ4Page; }

void launch_kv_q4_store_batch(uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* pos0,
                              const int32_t* row_off, int n_sess, int n_rows, int layer, int nb, const float* k,
                              const float* v, nova_stream_t s) {
    StoreArgs a{row_args(pool, tables, table_stride, pos0, row_off, n_sess, n_rows, layer, nb), nullptr, 0};
    NOVA_REQUIRE(k && v && aligned16(k) && aligned16(v));
    if (n_rows == 0) return;
    a.k = k;
    a.v = v;
    hipLaunchKernelGGL((q4_store_kernel<false, kRopeApart4>), dim3(store_wgs<false>(a)), dim3(QT), 0,
                       reinterpret_cast<hipStream_t>(s), a);
    NOVA_LAUNCHED();
}

void launch_rope_rows_kv_q4_store_batch(const float* q, const float* k, const float* v, const float* cs, const float* sn,
                                        int rot_dim, int beside, uint8_t* pool, const int32_t* tables, int table_stride,
                                        const int32_t* n_past, const int32_t* row_off, int n_sess, int n_rows, int layer,
                                        int nb, float* q_out, nova_stream_t s) {
    StoreArgs a{row_args(pool, tables, table_stride, n_past, row_off, n_sess, n_rows, layer, nb), q, rot_dim};
    NOVA_REQUIRE(q && k && v && cs && sn && q_out);
    NOVA_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(cs) && aligned16(sn) && aligned16(q_out));
    NOVA_REQUIRE(rot_dim >= 2 && rot_dim <= HD && rot_dim % 2 == 0);
    if (n_rows == 0) return;
    a.q = q_out;
    a.k = k;
    a.v = v;
    a.cs = cs;
    a.sn = sn;
    rope_forms(rot_dim, beside != 0, [&](auto form) {
        hipLaunchKernelGGL((q4_store_kernel<true, decltype(form)::value>), dim3(store_wgs<true>(a)), dim3(QT), 0,
                           reinterpret_cast<hipStream_t>(s), a);
        NOVA_LAUNCHED();
    });
}

void launch_kv_q4_load_batch(const uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* pos0,
                             const int32_t* row_off, int n_sess, int n_rows, int layer, int nb, float* k, float* v,
                             nova_stream_t s) {
    RowArgs a = row_args(const_cast<uint8_t*>(pool), tables, table_stride, pos0, row_off, n_sess, n_rows, layer, nb);
    NOVA_REQUIRE(k && v && aligned16(k) && aligned16(v));
    if (n_rows == 0) return;
    a.k_out = k;
    a.v_out = v;
    hipLaunchKernelGGL(q4_load_kernel, dim3(page_bound(a), NKV), dim3(QT), 0, reinterpret_cast<hipStream_t>(s), a);
    NOVA_LAUNCHED();
}

void launch_kv_q4_cow_apply(uint8_t* pool, int nb, int32_t* tables_dev, const nova_cow_op* ops, int n_ops,
                            nova_stream_t s) {
    cow_apply<kQ4Page>(pool, nb, tables_dev, ops, n_ops, reinterpret_cast<hipStream_t>(s));
}

void launch_kv_q4_zero_pages(uint8_t* pool, int nb, const int32_t* pages, int n_pages, nova_stream_t s) {
    zero_pages<kQ4Page>(pool, nb, pages, n_pages, reinterpret_cast<hipStream_t>(s));
}

}  // extern "C"
