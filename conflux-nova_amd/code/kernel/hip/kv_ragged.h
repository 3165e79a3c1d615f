// kv_ragged.h -- rows of a ragged batch and pages of a block table, as every call over
// quantised pages takes them.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

#include "model.h"

namespace nova {

// Rows of a ragged call: session i owns rows [off[i], off[i+1]) of the flat
// arrays, or n rows each where there are no offsets.  Offsets come from device
// memory, so they are held inside [0, n_rows].
struct RaggedRows {
    const int32_t* off;        // device [n_sess + 1] or null
    int uniform;               // rows per session without offsets
    int n_rows;
};

__device__ __forceinline__ int row_first(const RaggedRows& r, int i) {
    return r.off ? min(max(r.off[i], 0), r.n_rows) : i * r.uniform;
}
__device__ __forceinline__ int row_count(const RaggedRows& r, int i) {
    return r.off ? max(row_first(r, i + 1) - row_first(r, i), 0) : r.uniform;
}

// record of logical page pg: table entries outside the pool read page 0, so
// that no address leaves it
__device__ __forceinline__ int page_or_0(const int32_t* table, int pg, int nb) {
    const int p = table[pg];
    return (unsigned)p < (unsigned)nb ? p : 0;
}

// sum over lanes 0..l of a whole wave
__device__ __forceinline__ int scan_incl(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // row 0 -> 1, 2 -> 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // rows 0, 1 -> 2, 3
    return v;
}

}  // namespace nova
