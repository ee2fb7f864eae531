// Quantising a row of the 4-bit cache by 16 lanes (gfx950); the store (kv4.hip) and the
// fused q/k norm + RoPE + store (fused.hip) share it.  Format: kv4.h; the rule: kv4.hip.
#pragma once

#include "kv4.h"

namespace aac {
namespace kv4 {

// dpp_ctrl: lane i takes lane i + 4, 8, 12 of its 16 (0 past the last)
constexpr int kDppRowShl4 = 0x104, kDppRowShl8 = 0x108, kDppRowShl12 = 0x10C;

// The scale byte of 32 elements whose largest is a (bits without the sign), and the scale.
__device__ __forceinline__ u32 scale_byte(u32 a) {
  return a >= 0x7f800000u ? 255u : (u32)min(max((int)((a + 0x200000u) >> 23) - 2, 2), 252);
}
template <int CTRL> __device__ __forceinline__ u32 dpp_umax(u32 a) {
  return max(a, (u32)__builtin_amdgcn_update_dpp(0, (int)a, CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ u32 bits_of(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The 16-byte piece of a row that a lane holds, or two of an fp32 row.  16-bit types: eight
// dims, 8 l .. 8 l + 7 of lane l, four lanes a scale.  fp32: 4 l .. and 64 + 4 l .., so
// that the lanes' 16 bytes lie side by side in each access; eight lanes a scale.
template <Dt DT> struct Piece {
  u32x4 w;
};
template <> struct Piece<Dt::FP32> {
  f32x4 a, b;
};

// Quantises a row and writes its codes and scales.  The 16-bit types stay as they are:
// their bit patterns, without the sign, are in order of size, two in an instruction, and
// the conversion takes them in pairs (unpacked to floats first 4,096 tokens of 8 heads
// take 4.6 us against 4.4, and 16,000 in the fused store 44.0 against 42.8).
template <Dt DT>
__device__ __forceinline__ void write_row(const Piece<DT>& x, int l, unsigned char* codes, u32* scales) {
  u32 s4;
  if constexpr (DT == Dt::FP32) {
    u32 a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a = max(a, bits_of(x.a[i]));
      b = max(b, bits_of(x.b[i]));
    }
    a = scale_byte(dpp_umax<kDppRowHalfMirror>(dpp_umax<kDppQuadXor2>(dpp_umax<kDppQuadXor1>(a))));
    b = scale_byte(dpp_umax<kDppRowHalfMirror>(dpp_umax<kDppQuadXor2>(dpp_umax<kDppQuadXor1>(b))));
    const float sa = __uint_as_float(a << 23), sb = __uint_as_float(b << 23);
    u32 w = 0, z = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x.a[0], x.a[1], sa, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x.a[2], x.a[3], sa, 1);
    z = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(z, x.b[0], x.b[1], sb, 0);
    z = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(z, x.b[2], x.b[3], sb, 1);
    *reinterpret_cast<u16*>(codes + 2 * l) = a == 255u ? 0 : (u16)w;
    *reinterpret_cast<u16*>(codes + 32 + 2 * l) = b == 255u ? 0 : (u16)z;
    const u32 both = a | b << 16;  // scales 0 and 2 from lane 0, 1 and 3 from lane 8
    s4 = both | (u32)__builtin_amdgcn_update_dpp(0, (int)both, kDppRowShl8, 0xF, 0xF, true) << 8;
  } else {
    typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32 mag = x.w[i] & 0x7fff7fffu;
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, mag));
    }
    u32 a = max((u32)m[0], (u32)m[1]);
    a = dpp_umax<kDppQuadXor2>(dpp_umax<kDppQuadXor1>(a));
    if constexpr (DT == Dt::BF16) a = scale_byte(a << 16);
    else a = scale_byte(__float_as_uint((float)__builtin_bit_cast(_Float16, (u16)a)));
    const float s = __uint_as_float(a << 23);
    u32 w = 0;
#define AAC_CVT(i)                                                                                              \
  {                                                                                                             \
    const u32 pair = x.w[i];                                                                                    \
    if constexpr (DT == Dt::BF16)                                                                               \
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, pair), s, i);               \
    else                                                                                                        \
      w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(f16x2, pair), s, i);                   \
  }
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
    AAC_CVT(0) AAC_CVT(1) AAC_CVT(2) AAC_CVT(3)
#undef AAC_CVT
    __builtin_nontemporal_store(a == 255u ? 0u : w, reinterpret_cast<u32*>(codes + 4 * l));
    // the four scales, from lanes 0, 4, 8 and 12
    s4 = a;
    s4 |= (u32)__builtin_amdgcn_update_dpp(0, (int)a, kDppRowShl4, 0xF, 0xF, true) << 8;
    s4 |= (u32)__builtin_amdgcn_update_dpp(0, (int)a, kDppRowShl8, 0xF, 0xF, true) << 16;
    s4 |= (u32)__builtin_amdgcn_update_dpp(0, (int)a, kDppRowShl12, 0xF, 0xF, true) << 24;
  }
  if (l == 0) *scales = s4;
}

// (block, row in it) of a cache row
__device__ __forceinline__ void split_row(const Cache& c, int64_t row, int64_t* blk, int* r) {
  if (row < 0x80000000ll) {  // (a 64-bit division is some 100 instructions)
    *blk = (u32)row / (u32)c.block_size;
  } else {
    *blk = row / c.block_size;
  }
  *r = (int)(row - *blk * c.block_size);
}

}  // namespace kv4
}  // namespace aac
