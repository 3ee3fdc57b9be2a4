// Page format of the paged latent cache held in 4 bits, shared by its kernels.
//
// A token is a 512-wide latent in 16 blocks of 32 e2m1 codes with one e8m0 scale each (the block
// format gfx950's scaled conversions take) and 64 rotary keys in bf16: 256 + 128 + 16 bytes where a
// bf16 row takes 1,152.  The rotary part stays in bf16: it is a ninth of the row and carries the
// positions.  A page of ps tokens (a power of two) holds
//     ps * 256 B codes | ps * 128 B rotary keys | ps * 16 B scales
// so a token's codes are two whole 128-byte lines and each part of a page is one run.
//
// Scale byte s stands for 2^(s - 127), the least power of two that holds the block's largest value
// within 6, between 2^-124 and 2^125 (every held value is then zero or a normal bf16 number; larger
// values saturate at 1.5 * 2^127); 255 stands for a block in which an infinity or a NaN was written:
// all its 32 values read as NaN.
#pragma once

#include "common.h"

namespace paged {
constexpr int kLat = 512, kRope = 64, kRow = kLat + kRope;
constexpr int kCodeB = kLat / 2, kRopeB = kRope * 2, kScaleB = kLat / 32;
constexpr int kTokenB = kCodeB + kRopeB + kScaleB;  // 400
constexpr int kMaxPageShift = 10;
constexpr uint32_t kNanScale = 255;
constexpr int kLeastExp = -124, kMostExp = 125;

// log2 of a page size, -1 for one that is no power of two in [1, 1024]
inline int page_shift(int page_size) {
  for (int s = 0; s <= kMaxPageShift; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

// the addresses of slot's three parts (0 <= slot < n_pages << shift)
struct TokenAt {
  int64_t code, rope, scale;
};
__device__ __forceinline__ TokenAt token_at(int slot, int shift, int64_t page_stride) {
  const int off = slot & ((1 << shift) - 1);
  const int64_t base = static_cast<int64_t>(slot >> shift) * page_stride;
  return {base + off * kCodeB, base + (static_cast<int64_t>(kCodeB) << shift) + off * kRopeB,
          base + (static_cast<int64_t>(kCodeB + kRopeB) << shift) + off * kScaleB};
}

// the sums of v over lanes 0 .. l, by register moves between the lanes (six LDS-routed shuffles take 800 cycles)
template <typename Add>
__device__ __forceinline__ int wave_scan(int v, Add add) {
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8: within 16 lanes
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = add(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // lane 15 (47) to lanes 16-31 (48-63)
  return add(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));  // lane 31 to lanes 32-63
}
__device__ __forceinline__ int wave_scan(int v) {
  return wave_scan(v, [](int x, int y) { return x + y; });
}

// 8 codes (one dword, low nibble first) of a block with scale byte s as 8 bf16: the values are exact
__device__ __forceinline__ uint4 decode8(uint32_t codes, uint32_t s) {
  const float scale = __uint_as_float(s << 23);
  uint4 v;
  v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return v;
}
}  // namespace paged

// host checks of a pool of pages; the launch functions call them before anything else
int paged_check_pool(const char* what, const void* pages, int64_t page_stride, int n_pages, int page_size);
