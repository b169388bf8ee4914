// Layout of the paged latent cache and the element conversions its kernels share.
//
// A page holds 64 tokens of one layer.  bf16 pages are what kern_k3_mla_prep_head writes: 64 rows of 576 (512 latent
// columns, 64 rope columns).  MXFP8 pages hold the same rows as three planes, so that each plane of a page is one
// contiguous, 16-byte aligned run:
//     [    0, 32768)  64 x 512 E4M3 codes
//     [32768, 40960)  64 x 64 bf16: the rope columns, kept as they are (they carry positions; 128 of 1152 bytes)
//     [40960, 41984)  64 x 16 UE8M0 scale bytes, one per 32 codes
// 656 bytes per token against 1152.  Codes and scales are k3g_moe_quant's for the same 512 columns.
#pragma once
#include "k3g_device.cuh"

namespace k3g {

constexpr int kPageTokens = 64, kLatent = 512, kRopeCols = 64, kRow = kLatent + kRopeCols;   // 576
constexpr int kPageRope = kPageTokens * kLatent, kPageScales = kPageRope + kPageTokens * kRopeCols * 2;
constexpr int kMx8Page = kPageScales + kPageTokens * (kLatent / 32);                          // 41984 bytes
constexpr int kBf16Page = kPageTokens * kRow;                                                 // 36864 elements

// 2^(s - 127) as a pair of bf16: 0 is the subnormal 2^-127, 255 the format's NaN.
__device__ __forceinline__ unsigned ue8m0_pair(unsigned s) { return (s == 0 ? 0x0040u : s == 255 ? 0x7fffu : s << 7) * 0x10001u; }

// Four E4M3 codes times a power of two -> four bf16 in two words.  A code has four significant bits, so it is exact in f16 (which the
// conversion gives) and in bf16, and so is its product (but for the last bits of bf16 subnormals, rounded once).
__device__ __forceinline__ void mx8_to_bf16x4(unsigned codes, unsigned scale, unsigned& lo, unsigned& hi) {
  unsigned h0, h1;
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(h0), "=r"(h1) : "r"(codes));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0)), b = __half22float2(*reinterpret_cast<const __half2*>(&h1));
  lo = mul_bf2(pack_bf2(a.x, a.y), scale);
  hi = mul_bf2(pack_bf2(b.x, b.y), scale);
}

}  // namespace k3g
