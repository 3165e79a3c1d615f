// kv_q4.h -- the 4-bit page format and what its kernels share.
//
// A cached row x (128 values of one token and kv head, K or V) is held as 4-bit floating
// point codes c (two exponent bits, one of mantissa: 0, .5, 1, 1.5, 2, 3, 4, 6 for codes 0
// to 7, the sign in bit 3) with a power of two 2^e per 32 dims, value = c 2^e, e held as
// the byte e + 127: the block-scaled fp4 operand of gfx950's matrix instructions, so the
// score products take K from the page as it is.  A page of one layer is a record of
// kQ4Rec bytes per kv head, [layer][NB][NKV][kQ4Rec]:
//
//   K codes      token t, dim d at t * 64 + (d >> 1), the low half of the byte for even d
//   V codes      token t, dim d at kQ4VOff + (d >> 5) * 256 + (d & 15) * 16 + t, the low
//                half where bit 4 of d is clear
//   K exponents  token t, dims 32 j .. at kQ4KeOff + (t & 3) * 16 + j * 4 + (t >> 2)
//   V exponents  token t, dims 32 j .. at kQ4VeOff + j * 16 + t
//
// The layout is what attn_q4.hip reads, 16 B per lane with nothing to move afterwards.  A
// wave takes four pages; row 4p + i of its key block u is token 4u + i of page p, so K is
// 32 dims of one token per lane, and the four exponents that a lane needs for its four key
// blocks are one word, whose bytes the instructions select.  Lane (g, c) then holds the
// scores of all 16 tokens of page g for column c, and takes V as 16 tokens of two dims of
// one block of 32, which share their exponents.  All-zero memory is a valid page whose
// values are all zero; an exponent byte of 255 stands for NaN.
#pragma once
#include <cstdint>

#include "kv_ragged.h"
#include "model.h"

namespace nova {

constexpr int kQ4KBytes = Model::HD / 2 * kKvBlock;          // K codes of a record, and V codes
constexpr int kQ4VOff = kQ4KBytes;
constexpr int kQ4KeOff = 2 * kQ4KBytes;
constexpr int kQ4VeOff = kQ4KeOff + 4 * kKvBlock;
constexpr int kQ4Rec = kQ4VeOff + 4 * kKvBlock;              // 2176
constexpr int64_t kQ4Page = (int64_t)Model::NKV * kQ4Rec;    // one page of one layer
constexpr int kQ4Nan = 255;
// Exponent bytes that the quantiser makes, beside 0 and 255: 2^-100 to 2^96, so that sums of
// 2^21 products of weights (2^8 at most) and values stay inside fp32, and products of values with
// weights of 2^-24 and more above its subnormal numbers.
constexpr int kQ4LeastExp = 27, kQ4MostExp = 223;
static_assert(kQ4Rec == 2176, "documented record size");

}  // namespace nova
