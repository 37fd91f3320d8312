// The 4-bit form of a paged key/value cache, shared by its writes and reads
// (paged_rotary.hip) and its attention (seq_attn_fp4.h).
//
// Groups of 32 neighbouring dims are E2M1 elements (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
// negatives) with a scale byte b for 2^(b - 127), 255 for a group that holds an infinity
// or a NaN: a format that the conversions expand to 16 bits, scale and all, two elements at
// a time.
//
// The bytes of one page and key head, one after the other, with G = ceil(head_dim / 32)
// and S = page_size:
//   keys' codes [S, 16 G], values' codes [S, 16 G], keys' scales [S, 4], values' scales
//   [S, 4].
// Head by head, so that 16 tokens of a head are 1 KB in a row (128 dims) and every load
// of a wave fills whole memory lines; with the tokens of a page side by side the heads
// would share each line.  A head's scales of 16 tokens, keys and values, fill one line.
#pragma once

#include "dsa_common.h"

namespace fp4 {

constexpr int kGroup = 32;  // dims to a scale byte

// Exponents of the groups that a write makes: every element is a number of its type.
constexpr int kLowBf16 = -125, kHighBf16 = 125, kLowF16 = -23, kHighF16 = 13;

__host__ __device__ constexpr int groups_of(int head_dim) { return (head_dim + 31) / 32; }
__host__ __device__ constexpr int row_bytes(int groups) { return 32 * groups + 8; }

// Pages of up to 2^20 tokens, so that a page and head's bytes count in 32 bits.
constexpr int kMaxPage = 1 << 20;
inline bool bad_page_size(int32_t size) {
  return size < 16 || size > kMaxPage || (size & (size - 1)) != 0;
}

// Offsets within a page and head.
struct Layout {
  int32_t code_row, v_codes, k_scales, v_scales;
  __host__ __device__ Layout(int groups, int page_shift)
      : code_row(16 * groups),
        v_codes((16 * groups) << page_shift),
        k_scales((32 * groups) << page_shift),
        v_scales((32 * groups + 4) << page_shift) {}
};

// The float 2^(b - 127) as the conversions take it: its exponent field alone counts (0
// stands for 2^-127), and 255 makes NaN of every element.
__device__ __forceinline__ float scale_of(uint32_t b) { return __uint_as_float(b << 23); }

// Eight elements of a dword of codes (element 2 i: the low half of byte i).
__device__ __forceinline__ dsa_bf16x8 expand(uint32_t codes, float scale, __bf16) {
  const dsa_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  const dsa_bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  const dsa_bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  const dsa_bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return dsa_bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ dsa_f16x8 expand(uint32_t codes, float scale, _Float16) {
  const dsa_f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0);
  const dsa_f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1);
  const dsa_f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2);
  const dsa_f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3);
  return dsa_f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace fp4
