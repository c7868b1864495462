// The 8-bit paged cache: K and V held as int8 or float8 (e4m3) codes with one
// fp32 scale per block of 16 tokens and head; value = code * scale.
//
// Pages of n = 64 << k tokens hold all H kv heads of one sequence's tokens:
//   kpool  (P, H, n, d)         a token's codes in a row
//   vpool  (P, H, n / 16, d, 16) a block's tokens innermost, so that one coordinate's
//          16 codes are one load: tokens are the summed index of the value product
//   kscale / vscale (P, H, n / 16)
#pragma once

#include "qkv_common.h"

constexpr int kBlk = 16;  // tokens of a scale block

template <bool FP8>
constexpr float kTop = FP8 ? 448.f : 127.f;
constexpr float kScaleFloor = 0x1p-100f;  // of a block with a value other than 0

// Checks that the append, read and attention entry points share.
int qkv_kv8_check(int32_t fmt, int32_t num_pages, int32_t page_tokens, int32_t H, int32_t d);
