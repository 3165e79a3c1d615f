// attn_q8.hip -- attention over the 8-bit pages (kv_q8.h): one query token per
// session (decode), or a ragged chunk of new tokens per session, causally.
//
// o_h = sum_t softmax_t(q_h . k_t / sqrt(HD)) v_t, k_t = ks_t * code, v_t = vs_t * code,
// over keys [0, n_keys) or, for row r of a chunk, [0, n_past + r].
//
// One workgroup per (row, query head).  256 keys at a time: a thread forms one
// key's score, the workgroup their maximum and sum, and then each thread adds
// 128 keys to one head dim.  Everything is fp32.
#include <hip/hip_runtime.h>
#include <cstdint>

#include "check.h"
#include "kv_q8.h"
#include "model.h"
#include "nova_kernel.h"

namespace nova {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int NH = Model::NH, NKV = Model::NKV, HD = Model::HD, G = Model::G;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int AT = 256;

struct Q8Args {
    const float* q;            // [n_rows][NH][HD]
    const uint8_t* pool;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* n_keys;     // decode: keys of each session; chunk: its prefix
    Q8Rows rows;
    int causal;                // chunk: row r sees n_keys + r + 1 keys
    int n_sess;
    int layer;
    int nb;
    float* o;
};

__global__ void __launch_bounds__(AT) q8_attn_simple(Q8Args a) {
    __shared__ float s_q[HD], s_p[AT], s_red[AT / 64], s_o[HD];
    const int row = blockIdx.y, head = blockIdx.x, tid = threadIdx.x;
    int sess = row / max(a.rows.uniform, 1);
    if (a.rows.off) {
        int lo = 0, hi = a.n_sess;                       // the last session that starts at or before row
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (q8_row0(a.rows, mid) <= row) lo = mid;
            else hi = mid;
        }
        sess = lo;
    }
    const int at = row - q8_row0(a.rows, sess);
    if (at < 0 || at >= q8_count(a.rows, sess)) return;
    const int64_t most = a.table_stride * kKvBlock;
    int64_t n64 = (int64_t)a.n_keys[sess] + (a.causal ? at + 1 : 0);
    const int n = (int)(n64 < 0 ? 0 : n64 < most ? n64 : most);
    const int32_t* table = a.tables + sess * a.table_stride;
    if (tid < HD) s_q[tid] = a.q[((int64_t)row * NH + head) * HD + tid] * (kScale * kLog2e);
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc = 0.f;
    const int d = tid % HD, half = tid / HD;
    for (int base = 0; base < n; base += AT) {
        const int t = base + tid;
        float x = -INFINITY;
        if (t < n) {
            const int slot = t & kKvBlockMask;
            const uint8_t* rec = a.pool + ((int64_t)a.layer * a.nb + q8_phys(table, t >> kKvBlockShift, a.nb)) * kQ8Page +
                                 (head / G) * kQ8Rec;
            const int8_t* k = reinterpret_cast<const int8_t*>(rec) + (slot >> 2) * 512 + (slot & 3) * 16;
            x = 0.f;
            for (int e = 0; e < HD; ++e) x += s_q[e] * (float)k[(e >> 4) * 64 + (e & 15)];
            x *= *reinterpret_cast<const float*>(rec + kQ8KsOff + 4 * slot);
        }
        float mx = x;
        for (int o = 32; o; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        if ((tid & 63) == 0) s_red[tid >> 6] = mx;
        __syncthreads();
        mx = m;
        for (int w = 0; w < AT / 64; ++w) mx = fmaxf(mx, s_red[w]);
        const float w = t < n ? __builtin_amdgcn_exp2f(x - mx) : 0.f;
        s_p[tid] = w;
        __syncthreads();
        const float corr = m == mx ? 1.f : __builtin_amdgcn_exp2f(m - mx);
        m = mx;
        l = l * corr + w;                                // this thread's keys
        acc *= corr;
        float part = 0.f;
        for (int u = half * (AT / 2); u < (half + 1) * (AT / 2) && base + u < n; ++u) {
            const int key = base + u, slot = key & kKvBlockMask;
            const uint8_t* rec = a.pool +
                                 ((int64_t)a.layer * a.nb + q8_phys(table, key >> kKvBlockShift, a.nb)) * kQ8Page +
                                 (head / G) * kQ8Rec;
            part += s_p[u] * *reinterpret_cast<const float*>(rec + kQ8VsOff + 4 * slot) *
                    (float)(int8_t)rec[kQ8VOff + d * kKvBlock + slot];
        }
        acc += part;
        __syncthreads();
    }
    if (half == 1) s_o[d] = acc;
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o, 64);
    if ((tid & 63) == 0) s_red[tid >> 6] = l;
    __syncthreads();
    l = 0.f;
    for (int w = 0; w < AT / 64; ++w) l += s_red[w];
    if (half == 0) a.o[((int64_t)row * NH + head) * HD + d] = n > 0 ? (acc + s_o[d]) / l : 0.f;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

Q8Args attn_args(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride, const int32_t* n_keys,
                 int n_sess, int layer, int nb, float* o) {
    NOVA_REQUIRE(q && pool && tables && n_keys && o);
    NOVA_REQUIRE(aligned16(q) && aligned16(pool) && aligned16(o));
    NOVA_REQUIRE(layer >= 0 && layer < Model::L && nb > 0 && table_stride > 0 && table_stride <= (1 << 27));
    Q8Args a{};
    a.q = q;
    a.pool = pool;
    a.tables = tables;
    a.table_stride = table_stride;
    a.n_keys = n_keys;
    a.n_sess = n_sess;
    a.layer = layer;
    a.nb = nb;
    a.o = o;
    return a;
}

}  // namespace
}  // namespace nova

using namespace nova;

extern "C" {

size_t attn_decode_q8_workspace_bytes(int n_sess) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535);
    return 16;
}

size_t attn_chunk_q8_workspace_bytes(int n_sess, int n_rows, int max_q) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && n_rows >= 0 && max_q >= 0 && max_q <= n_rows);
    return 16;
}

void launch_attn_decode_q8_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                 const int32_t* n_keys, int n_sess, int layer, int nb, float* o, void* workspace,
                                 nova_stream_t s) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535);
    Q8Args a = attn_args(q, pool, tables, table_stride, n_keys, n_sess, layer, nb, o);
    NOVA_REQUIRE(workspace && aligned16(workspace));
    a.rows = Q8Rows{nullptr, 1, n_sess};
    hipLaunchKernelGGL(q8_attn_simple, dim3(NH, n_sess), dim3(AT), 0, reinterpret_cast<hipStream_t>(s), a);
    NOVA_LAUNCHED();
}

void launch_attn_chunk_q8_batch(const float* q, const uint8_t* pool, const int32_t* tables, int table_stride,
                                const int32_t* n_past, const int32_t* row_off, int n_sess, int n_rows, int max_q,
                                int layer, int nb, float* o, void* workspace, nova_stream_t s) {
    NOVA_REQUIRE(n_sess >= 1 && n_sess <= 65535 && n_rows >= 0 && n_rows <= 65535);
    NOVA_REQUIRE(max_q >= 0 && max_q <= n_rows);
    NOVA_REQUIRE(row_off || n_rows % n_sess == 0);
    Q8Args a = attn_args(q, pool, tables, table_stride, n_past, n_sess, layer, nb, o);
    NOVA_REQUIRE(workspace && aligned16(workspace));
    if (n_rows == 0) return;
    a.rows = Q8Rows{row_off, n_rows / n_sess, n_rows};
    a.causal = 1;
    hipLaunchKernelGGL(q8_attn_simple, dim3(NH, n_rows), dim3(AT), 0, reinterpret_cast<hipStream_t>(s), a);
    NOVA_LAUNCHED();
}

}  // extern "C"
