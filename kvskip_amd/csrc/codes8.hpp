// Codes of a cache held in 8 bits as operands of fp16 matrix products: conversions and the register layouts of a 64-token
// block's keys and values (the passes of attn_decode8.hip and attend.hip).
#pragma once

#include "attn_common.hpp"

namespace kvs {
namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// Four codes of a dword as fp16: codes 0, 1 and codes 2, 3.
template <bool I8>
__device__ __forceinline__ u32x2 widen4(uint32_t w) {
  uint32_t lo, hi;
  if constexpr (I8) {
    const uint32_t u = w ^ 0x80808080u;  // x + 128
    const f16x2_t off = {-1152.f16, -1152.f16};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
  } else {
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
  }
  return u32x2{lo, hi};
}

__device__ __forceinline__ u32x2 bload8(rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_amdgcn_raw_buffer_load_b64(r, static_cast<int>(voff), static_cast<int>(soff), BUF_NT);
}

// Sizes of a block's registers: K as 16-byte chunks of a row (lane r = lane % 16, j = lane / 16 holds bytes 16 j + 64 c
// of row 16 nt + r, which are k-steps 2 c and 2 c + 1 of the scores' products; q is laid out alike), V as 8 bytes of a
// row (D 128: a 16-lane group loads one row; D 64: two, and lanes c and c ^ 8 exchange halves).
template <int D>
struct Lay8 {
  static constexpr int KC = D / 64;
  static constexpr int KS = D / 32;
  static constexpr int VN = BLK * D / (WAVE * 8);
  static constexpr int VD = D / 16;
};

template <int D>
__device__ __forceinline__ void load_k8(u32x4 (&kr)[4][Lay8<D>::KC], rsrc_t r, uint32_t koff, uint32_t st) {
#pragma unroll
  for (int nt = 0; nt < 4; ++nt)
#pragma unroll
    for (int c = 0; c < Lay8<D>::KC; ++c) kr[nt][c] = bload16<BUF_NT>(r, koff + 64 * c, 16 * nt * st);
}

template <int D>
__device__ __forceinline__ void load_v8(u32x2 (&vr)[Lay8<D>::VN], rsrc_t r, uint32_t voff, uint32_t st) {
#pragma unroll
  for (int i = 0; i < Lay8<D>::VN; ++i) {
    const int t = D == 128 ? mf_tok(i / 4, i % 4, 0) : mf_tok(i / 2, 2 * (i % 2), 0);
    vr[i] = bload8(r, voff, t * st);
  }
}

// Dword d (4 dims) of tokens (nt, i) and (nt, i + 1), i even, of this lane's column.
template <int D>
__device__ __forceinline__ void v_pair8(const u32x2 (&vr)[Lay8<D>::VN], int nt, int i, int d, bool up, uint32_t& a,
                                        uint32_t& c) {
  if constexpr (D == 128) {
    a = vr[4 * nt + i][d];
    c = vr[4 * nt + i + 1][d];
  } else {  // up: lanes c >= 8, which loaded the second token's row
    const u32x2 x = vr[2 * nt + i / 2];
    const uint32_t other = dppu<DPP_ROR8>(up ? x.x : x.y);
    a = up ? other : x.x;
    c = up ? x.y : other;
  }
}

// 2^y in two factors, for y of which the whole may lie below or above what fp32 holds (2^-133 where a scale is 2^-126). The second
// is a whole power of two, so whole y stay exact.
struct Pow2 {
  float a, b;
  __device__ __forceinline__ explicit Pow2(float y) {
    const float k = fmaxf(rintf(0.5f * y), -1000.f);  // (y may be -infinity)
    a = fexp2(y - k), b = fexp2(k);
  }
};

// Two values as fp16, to nearest even, the first in the low half.
__device__ __forceinline__ uint32_t pack_h(float a, float b) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{a, b}), f16x2_t));
}

// (a, b) c + h as fp16, rounded once (v_fma_mixlo_f16, v_fma_mixhi_f16).
__device__ __forceinline__ uint32_t mix_h(float a, float b, float c, f16x2_t h) {
  return __builtin_bit_cast(uint32_t, f16x2_t{static_cast<_Float16>(fmaf(a, c, static_cast<float>(h.x))),
                                              static_cast<_Float16>(fmaf(b, c, static_cast<float>(h.y)))});
}

}  // namespace
}  // namespace kvs
