// kv_q8.h -- the 8-bit page format and what its kernels share.
//
// A cached row x (128 values of one token and kv head, K or V) is held as int8
// codes c with one fp32 scale s, value = c * s.  A page of one layer is a record
// of kQ8Rec bytes per kv head, [layer][NB][NKV][kQ8Rec]:
//
//   K codes   token t, dim d at (t >> 2) * 512 + (d >> 4) * 64 + (t & 3) * 16 + (d & 15)
//   V codes   token t, dim d at kQ8VOff + d * 16 + t
//   K scales  token t at kQ8KsOff + 4 t
//   V scales  token t at kQ8VsOff + 4 t
//
// The layout is what the matrix instructions of attn_q8.hip read, 16 B per lane
// with nothing to move afterwards.  The score product is K . Q^T over 64 dims
// at a time; a wave takes four pages, and row 4g + i of its key block kb is
// token 4 kb + i of page g.  Lane (g, c) then holds, after the four key blocks,
// the scores of all 16 tokens of page g for column c, in token order: which is
// how V^T . P^T wants them, with V as 16 tokens of one dim per lane.  Each load
// instruction of a wave covers 256 contiguous bytes of each page, and a record
// of one kv head is 33 whole 128 B lines.  All-zero memory is a valid page whose
// values are all zero.
#pragma once
#include <cstdint>

#include "model.h"

namespace nova {

constexpr int kQ8KBytes = Model::HD * kKvBlock;              // K codes of a record, and V codes
constexpr int kQ8VOff = kQ8KBytes;
constexpr int kQ8KsOff = 2 * kQ8KBytes;
constexpr int kQ8VsOff = kQ8KsOff + 4 * kKvBlock;
constexpr int kQ8Rec = kQ8VsOff + 4 * kKvBlock;              // 4224
constexpr int64_t kQ8Page = (int64_t)Model::NKV * kQ8Rec;    // one page of one layer
static_assert(kQ8Rec == 4224, "documented record size");

// Rows of a ragged call: session i owns rows [off[i], off[i+1]) of the flat
// arrays, or n rows each where there are no offsets.  Offsets come from device
// memory, so they are held inside [0, n_rows].
struct Q8Rows {
    const int32_t* off;        // device [n_sess + 1] or null
    int uniform;               // rows per session without offsets
    int n_rows;
};

__device__ __forceinline__ int q8_row0(const Q8Rows& r, int i) {
    return r.off ? min(max(r.off[i], 0), r.n_rows) : i * r.uniform;
}
__device__ __forceinline__ int q8_count(const Q8Rows& r, int i) {
    return r.off ? max(q8_row0(r, i + 1) - q8_row0(r, i), 0) : r.uniform;
}

// record of logical page pg: table entries outside the pool read page 0, so
// that no address leaves it
__device__ __forceinline__ int q8_phys(const int32_t* table, int pg, int nb) {
    const int p = table[pg];
    return (unsigned)p < (unsigned)nb ? p : 0;
}

}  // namespace nova
