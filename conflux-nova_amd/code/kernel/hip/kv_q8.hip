// kv_q8.hip -- 8-bit pages: quantise K and V as they are written (alone or with
// RoPE), read rows back, copy-on-write page copies and page clears.
//
// Quantiser, per row x of 128 values: a = max |x|, s = fp32(a / 127),
// c = the integer nearest to the exact quotient x / s (ties to even), so that
// |c| <= 127.  s is held to the largest number whose 127 s is finite (rounded up,
// it passes that for a next to the largest fp32 number), and an s below the
// smallest normal number counts as 0 (codes 0); a row with an infinity or a NaN
// gets the scale NaN (codes 0), so that it reads back as NaN and never as a
// finite value.  The quotient is formed as x * (1 / s), whose error is under
// 2^-15 of a code; where that lies within 2^-13 of the middle between two codes,
// the two sides are compared exactly (in double, x against (c + 1/2) s: 32
// significant bits, no rounding).
//
// Layout of the work: a workgroup takes one page of one session's call and one
// kv head, 16 lanes per token; lane j holds dims 4j..4j+3 and 64+4j..64+4j+3
// (16 B loads in address order, and RoPE's pairs meet in one lane).  V codes are
// stored dim by dim, 16 tokens together: a page that the call fills goes through
// LDS and leaves as 16 B per lane; a page written in part (a decode step's one
// token, a chunk's ends) is written byte by byte, so that the other tokens of
// the page stay as they are.
//
// All of it is movement, bound by HBM once the call is large and by the launch
// before that.  8 x 512 tokens of the 7B model, appended and read back (21.1 MB each),
// take 13.5 us in two launches, 3.1 TB/s, where a large copy moves 5.2 TB/s; RoPE and
// append of the same tokens (138 MB, the rotated queries most of it) 28 us, 4.9 TB/s.
// A decode step's 16 tokens, appended and read back, take 10 us, which is the calls
// and their launches.  64 page copies of the 7B model over all layers, 30 MB written
// from 4 donors, take 8.6 us, 3.7 TB/s, with the launch; one of the 1.5B model 8.3.
#include <hip/hip_runtime.h>
#include <cstdint>

#include "check.h"
#include "kv_q8.h"
#include "kv_rows.h"
#include "model.h"
#include "nova_kernel.h"
#include "rope_math.h"

namespace nova {
namespace {

constexpr int NH = Model::NH, NKV = Model::NKV, HD = Model::HD;
constexpr int HALF = HD / 2;
constexpr int kLanes = 16;                     // lanes per token
constexpr int QT = kKvBlock * kLanes;          // threads of a workgroup
static_assert(QT == 256 && kLanes * 8 == HD, "one page per workgroup, 8 dims per lane");

// the largest scale whose 127 * s is finite
constexpr float kMaxScale = 0x1.020406p+121f;

// scale of the row whose largest |x| has the bits `top` (infinities and NaN are
// the largest of all)
__device__ __forceinline__ float row_scale(uint32_t top) {
    const float s = fminf(__uint_as_float(top) / 127.0f, kMaxScale);
    if (top >= 0x7f800000u) return __builtin_nanf("");
    return s >= 1.17549435e-38f ? s : 0.f;
}

__device__ __forceinline__ int row_code(float x, float s, float inv) {
    const float q = x * inv;
    float r = __builtin_rintf(q);
    const float away = fabsf(q - r);               // exact: both are near and small
    if (away > 0.5f - 0x1p-13f) {
        // between codes f and f + 1: x against (f + 1/2) s, exactly
        const float f = __builtin_floorf(q);
        const double mid = ((double)f + 0.5) * (double)s, dx = (double)x;
        r = dx > mid ? f + 1.f : dx < mid ? f : 2.f * __builtin_rintf(0.5f * (f + 0.5f));
    }
    return (int)r;
}

// codes of a lane's 8 dims, packed four to a word; the scale is returned
__device__ __forceinline__ float quantise(const f4 a, const f4 b, uint32_t& w0, uint32_t& w1) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        top = max(top, __float_as_uint(a[e]) & 0x7fffffffu);
        top = max(top, __float_as_uint(b[e]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, kLanes));
    const float s = row_scale(top);
    w0 = w1 = 0;
    if (s > 0.f) {
        const float inv = 1.0f / s;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w0 |= (uint32_t)(row_code(a[e], s, inv) & 255) << (8 * e);
            w1 |= (uint32_t)(row_code(b[e], s, inv) & 255) << (8 * e);
        }
    }
    return s;
}

// grid: x = pages of the call (an upper bound), y = kv heads, then (RoPE) query
// heads, whose rows are rotated in place
template <bool kRope>
__global__ void __launch_bounds__(QT) q8_store_kernel(RowArgs a) {
    const PageItem it = page_item(a, blockIdx.x);
    if (it.sess < 0) return;
    const int t = threadIdx.x / kLanes, j = threadIdx.x % kLanes;
    const int pos = it.page * kKvBlock + t;
    const int first = max(it.pos0 - it.page * kKvBlock, 0);                   // tokens [first, last) of the page
    const int last = min(it.pos0 + it.n - it.page * kKvBlock, kKvBlock);
    const bool real = t >= first && t < last;
    const int64_t row = it.row0 + pos - it.pos0;
    f4 c{}, s{};
    if constexpr (kRope) {
        if (real) {
            c = *reinterpret_cast<const f4*>(a.cs + (int64_t)pos * HALF + 4 * j);
            s = *reinterpret_cast<const f4*>(a.sn + (int64_t)pos * HALF + 4 * j);
        }
        if ((int)blockIdx.y >= NKV) {                                        // a query head
            if (!real) return;
            float* x = a.q + (row * NH + blockIdx.y - NKV) * HD + 4 * j;
            f4 x0 = *reinterpret_cast<const f4*>(x), x1 = *reinterpret_cast<const f4*>(x + HALF);
            f4 y0, y1;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float p, r;
                rope_rotate(x0[e], x1[e], c[e], s[e], p, r);
                y0[e] = p;
                y1[e] = r;
            }
            *reinterpret_cast<f4*>(x) = y0;
            *reinterpret_cast<f4*>(x + HALF) = y1;
            return;
        }
    }
    const int head = blockIdx.y;
    f4 x0{}, x1{}, y0{}, y1{};                                               // the rows, requested beside the table entry
    if (real) {
        const float* src = a.k + (row * NKV + head) * HD + 4 * j;
        x0 = *reinterpret_cast<const f4*>(src);
        x1 = *reinterpret_cast<const f4*>(src + HALF);
        src = a.v + (row * NKV + head) * HD + 4 * j;
        y0 = *reinterpret_cast<const f4*>(src);
        y1 = *reinterpret_cast<const f4*>(src + HALF);
    }
    const int phys = a.tables[it.sess * a.table_stride + it.page];
    if ((unsigned)phys >= (unsigned)a.nb) return;                            // no such page: nothing is written
    uint8_t* rec = a.pool + ((int64_t)a.layer * a.nb + phys) * kQ8Page + head * kQ8Rec;
    uint32_t v0 = 0, v1 = 0;
    if (real) {
        if constexpr (kRope) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float p, r;
                rope_rotate(x0[e], x1[e], c[e], s[e], p, r);
                x0[e] = p;
                x1[e] = r;
            }
        }
        uint32_t k0, k1;
        const float ks = quantise(x0, x1, k0, k1);
        uint8_t* dk = rec + (t >> 2) * 512 + (j >> 2) * 64 + (t & 3) * 16 + (j & 3) * 4;
        *reinterpret_cast<uint32_t*>(dk) = k0;
        *reinterpret_cast<uint32_t*>(dk + 256) = k1;
        const float vs = quantise(y0, y1, v0, v1);
        if (j == 0) {
            *reinterpret_cast<float*>(rec + kQ8KsOff + 4 * t) = ks;
            *reinterpret_cast<float*>(rec + kQ8VsOff + 4 * t) = vs;
        }
    }
    if (first == 0 && last == kKvBlock) {                                    // uniform over the workgroup
        __shared__ __attribute__((aligned(16))) uint8_t s_v[HD * kKvBlock];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s_v[(4 * j + e) * kKvBlock + t] = (uint8_t)(v0 >> (8 * e));
            s_v[(HALF + 4 * j + e) * kKvBlock + t] = (uint8_t)(v1 >> (8 * e));
        }
        __syncthreads();
        if (threadIdx.x < HD)
            *reinterpret_cast<u4*>(rec + kQ8VOff + 16 * threadIdx.x) = *reinterpret_cast<const u4*>(s_v + 16 * threadIdx.x);
    } else if (real) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            rec[kQ8VOff + (4 * j + e) * kKvBlock + t] = (uint8_t)(v0 >> (8 * e));
            rec[kQ8VOff + (HALF + 4 * j + e) * kKvBlock + t] = (uint8_t)(v1 >> (8 * e));
        }
    }
}

__device__ __forceinline__ f4 values(uint32_t w, float s) {
    f4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (float)(int8_t)(w >> (8 * e)) * s;
    return y;
}

// the reverse: c * s, rounded once
__global__ void __launch_bounds__(QT) q8_load_kernel(RowArgs a) {
    const PageItem it = page_item(a, blockIdx.x);
    if (it.sess < 0) return;
    const int t = threadIdx.x / kLanes, j = threadIdx.x % kLanes;
    const int first = max(it.pos0 - it.page * kKvBlock, 0);
    const int last = min(it.pos0 + it.n - it.page * kKvBlock, kKvBlock);
    const int head = blockIdx.y;
    const int phys = page_or_0(a.tables + it.sess * a.table_stride, it.page, a.nb);
    const uint8_t* rec = a.pool + ((int64_t)a.layer * a.nb + phys) * kQ8Page + head * kQ8Rec;
    // every read of the record goes out before the first wait; V's codes, dim by dim
    // in the page, are read 16 B per lane and turned in LDS (reading them byte by
    // byte instead: 9.6 us for 8 x 512 rows of the 7B model, so 6.4)
    const uint8_t* pk = rec + (t >> 2) * 512 + (j >> 2) * 64 + (t & 3) * 16 + (j & 3) * 4;
    const uint32_t k0 = *reinterpret_cast<const uint32_t*>(pk), k1 = *reinterpret_cast<const uint32_t*>(pk + 256);
    const float ks = *reinterpret_cast<const float*>(rec + kQ8KsOff + 4 * t);
    const float vs = *reinterpret_cast<const float*>(rec + kQ8VsOff + 4 * t);
    __shared__ __attribute__((aligned(16))) uint8_t s_v[HD * kKvBlock];
    if (threadIdx.x < HD)
        *reinterpret_cast<u4*>(s_v + 16 * threadIdx.x) = *reinterpret_cast<const u4*>(rec + kQ8VOff + 16 * threadIdx.x);
    __syncthreads();
    if (t < first || t >= last) return;
    const int64_t row = it.row0 + it.page * kKvBlock + t - it.pos0;
    uint32_t v0 = 0, v1 = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v0 |= (uint32_t)s_v[(4 * j + e) * kKvBlock + t] << (8 * e);
        v1 |= (uint32_t)s_v[(HALF + 4 * j + e) * kKvBlock + t] << (8 * e);
    }
    float* k = a.k_out + (row * NKV + head) * HD + 4 * j;
    float* v = a.v_out + (row * NKV + head) * HD + 4 * j;
    *reinterpret_cast<f4*>(k) = values(k0, ks);
    *reinterpret_cast<f4*>(k + HALF) = values(k1, ks);
    *reinterpret_cast<f4*>(v) = values(v0, vs);
    *reinterpret_cast<f4*>(v + HALF) = values(v1, vs);
}

}  // namespace
}  // namespace nova

using namespace nova;

extern "C" {

size_t kv_q8_page_bytes(void) { return (size_t)kQ8Page; }

void launch_kv_q8_store_batch(uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* pos0,
                              const int32_t* row_off, int n_sess, int n_rows, int layer, int nb, const float* k,
                              const float* v, nova_stream_t s) {
    RowArgs a = row_args(pool, tables, table_stride, pos0, row_off, n_sess, n_rows, layer, nb);
    NOVA_REQUIRE(k && v && aligned16(k) && aligned16(v));
    if (n_rows == 0) return;
    a.k = k;
    a.v = v;
    hipLaunchKernelGGL(q8_store_kernel<false>, dim3(page_bound(a), NKV), dim3(QT), 0, reinterpret_cast<hipStream_t>(s),
                       a);
    NOVA_LAUNCHED();
}

void launch_rope_kv_q8_store_batch(float* q, const float* k, const float* v, const float* cs, const float* sn,
                                   uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* n_past,
                                   const int32_t* row_off, int n_sess, int n_rows, int layer, int nb,
                                   nova_stream_t s) {
    RowArgs a = row_args(pool, tables, table_stride, n_past, row_off, n_sess, n_rows, layer, nb);
    NOVA_REQUIRE(q && k && v && cs && sn);
    NOVA_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(cs) && aligned16(sn));
    if (n_rows == 0) return;
    a.q = q;
    a.k = k;
    a.v = v;
    a.cs = cs;
    a.sn = sn;
    hipLaunchKernelGGL(q8_store_kernel<true>, dim3(page_bound(a), NKV + NH), dim3(QT), 0,
                       reinterpret_cast<hipStream_t>(s), a);
    NOVA_LAUNCHED();
}

void launch_kv_q8_load_batch(const uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* pos0,
                             const int32_t* row_off, int n_sess, int n_rows, int layer, int nb, float* k, float* v,
                             nova_stream_t s) {
    RowArgs a = row_args(const_cast<uint8_t*>(pool), tables, table_stride, pos0, row_off, n_sess, n_rows, layer, nb);
    NOVA_REQUIRE(k && v && aligned16(k) && aligned16(v));
    if (n_rows == 0) return;
    a.k_out = k;
    a.v_out = v;
    hipLaunchKernelGGL(q8_load_kernel, dim3(page_bound(a), NKV), dim3(QT), 0, reinterpret_cast<hipStream_t>(s), a);
    NOVA_LAUNCHED();
}

void launch_kv_q8_cow_apply(uint8_t* pool, int nb, int32_t* tables_dev, const nova_cow_op* ops, int n_ops,
                            nova_stream_t s) {
    cow_apply<kQ8Page>(pool, nb, tables_dev, ops, n_ops, reinterpret_cast<hipStream_t>(s));
}

void launch_kv_q8_zero_pages(uint8_t* pool, int nb, const int32_t* pages, int n_pages, nova_stream_t s) {
    zero_pages<kQ8Page>(pool, nb, pages, n_pages, reinterpret_cast<hipStream_t>(s));
}

}  // extern "C"
