// rope_rows.h -- the rotation of one row by its own angles, shared by the kernels that
// apply it: the first `rot` dims of a head turn in pairs, half of them apart (dims i and
// i + rot/2) or side by side (2i and 2i + 1), by c[i] and s[i]; dims from rot on stay.
#pragma once
#include <hip/hip_runtime.h>
#include <type_traits>

#include "model.h"
#include "rope_math.h"

namespace nova {
namespace {

typedef float rope_f4 __attribute__((ext_vector_type(4)));

// How a row's pairs are walked: by fours where every group of four is aligned, else one by one.
enum RopeForm { kRopeApart4, kRopeApart1, kRopeBeside4, kRopeBeside1 };

__host__ __device__ __forceinline__ constexpr RopeForm rope_form(int rot, bool beside) {
    return beside ? (rot % 4 == 0 ? kRopeBeside4 : kRopeBeside1) : (rot % 8 == 0 ? kRopeApart4 : kRopeApart1);
}

// Units of a head: what one lane does at a time.  A unit reads what it writes and nothing
// else, so a row may be turned in place.
template <RopeForm kForm>
__device__ __forceinline__ int rope_units(int rot) {
    constexpr int HD = Model::HD;
    if constexpr (kForm == kRopeApart4) return rot / 8 + (HD - rot) / 4;
    else if constexpr (kForm == kRopeBeside4) return HD / 4;
    else return HD / 2;
}

// unit u of a head's row x -> y; c, s: the row's angles
template <RopeForm kForm>
__device__ __forceinline__ void rope_unit(const float* x, float* y, const float* c, const float* s, int rot, int u) {
    const int half = rot / 2;
    if constexpr (kForm == kRopeApart4) {
        if (u >= rot / 8) {
            const int d = rot + 4 * (u - rot / 8);
            *reinterpret_cast<rope_f4*>(y + d) = *reinterpret_cast<const rope_f4*>(x + d);
            return;
        }
        const int i = 4 * u;
        const rope_f4 x0 = *reinterpret_cast<const rope_f4*>(x + i), x1 = *reinterpret_cast<const rope_f4*>(x + half + i);
        const rope_f4 cc = *reinterpret_cast<const rope_f4*>(c + i), ss = *reinterpret_cast<const rope_f4*>(s + i);
        rope_f4 y0, y1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float a, b;
            rope_rotate(x0[e], x1[e], cc[e], ss[e], a, b);
            y0[e] = a;
            y1[e] = b;
        }
        *reinterpret_cast<rope_f4*>(y + i) = y0;
        *reinterpret_cast<rope_f4*>(y + half + i) = y1;
    } else if constexpr (kForm == kRopeBeside4) {
        const int d = 4 * u;
        rope_f4 z = *reinterpret_cast<const rope_f4*>(x + d);
        if (d < rot) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                float a, b;
                rope_rotate(z[e], z[e + 1], c[d / 2 + e / 2], s[d / 2 + e / 2], a, b);
                z[e] = a;
                z[e + 1] = b;
            }
        }
        *reinterpret_cast<rope_f4*>(y + d) = z;
    } else {
        // pair u of the head, those of the dims that stay behind the turning ones
        const bool turns = u < half;
        const int d0 = turns && kForm == kRopeApart1 ? u : 2 * u, d1 = turns && kForm == kRopeApart1 ? u + half : 2 * u + 1;
        float a = x[d0], b = x[d1];
        if (turns) {
            float ya, yb;
            rope_rotate(a, b, c[u], s[u], ya, yb);
            a = ya;
            b = yb;
        }
        y[d0] = a;
        y[d1] = b;
    }
}

// dims 8 j .. 8 j + 7 of the turned row, from the row as it is
template <RopeForm kForm>
__device__ __forceinline__ void rope_dims8(const float* x, const float* c, const float* s, int rot, int j, float (&y)[8]) {
    const int half = rot / 2;
    if constexpr (kForm == kRopeApart4) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {                     // four dims on one side of every border
            const int d = 8 * j + e;
            const rope_f4 mine = *reinterpret_cast<const rope_f4*>(x + d);
            const bool low = d < half, turns = d < rot;
            const int i = low ? d : d - half, o = low ? d + half : d - half;
            rope_f4 other = mine, cc{}, ss{};
            if (turns) {
                other = *reinterpret_cast<const rope_f4*>(x + o);
                cc = *reinterpret_cast<const rope_f4*>(c + i);
                ss = *reinterpret_cast<const rope_f4*>(s + i);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float a, b;
                rope_rotate(low ? mine[k] : other[k], low ? other[k] : mine[k], cc[k], ss[k], a, b);
                y[e + k] = !turns ? mine[k] : low ? a : b;
            }
        }
    } else if constexpr (kForm == kRopeApart1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int d = 8 * j + e;
            y[e] = x[d];
            if (d < rot) {
                const bool low = d < half;
                const int i = low ? d : d - half;
                float a, b;
                rope_rotate(x[i], x[i + half], c[i], s[i], a, b);
                y[e] = low ? a : b;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const int d = 8 * j + e;
            y[e] = x[d];
            y[e + 1] = x[d + 1];
            if (d < rot) {
                float a, b;
                rope_rotate(y[e], y[e + 1], c[d / 2], s[d / 2], a, b);
                y[e] = a;
                y[e + 1] = b;
            }
        }
    }
}

// f(std::integral_constant<RopeForm, ...>) for the form of a call
template <class F>
void rope_forms(int rot, bool beside, F&& f) {
    switch (rope_form(rot, beside)) {
        case kRopeApart4: f(std::integral_constant<RopeForm, kRopeApart4>{}); break;
        case kRopeApart1: f(std::integral_constant<RopeForm, kRopeApart1>{}); break;
        case kRopeBeside4: f(std::integral_constant<RopeForm, kRopeBeside4>{}); break;
        case kRopeBeside1: f(std::integral_constant<RopeForm, kRopeBeside1>{}); break;
    }
}

}  // namespace
}  // namespace nova
