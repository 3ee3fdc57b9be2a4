// Products of e4m3 activations and e4m3 weights with block scales, dense and grouped by rows.
// No counterpart in the reference, whose products are bf16.
//
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} x[m, k] w[n, k]
//
// A block of 16 features x 16 tokens is summed from zero by matrix instructions, multiplied by sx sw on the VALU
// and added to the fp32 accumulator.  Features are the A operand, tokens the B operand, so that a lane holds one
// token's sums of neighbouring features: one factor a lane and block, and stores along the row.  Within a block both
// operands may order k as they like: lane group g of 16 takes the 16-byte pieces g and g + 4 of a row's 128 bytes.
//
// Two forms of a block's sum.  bf16 results take v_mfma_f32_16x16x128_f8f6f4 (32 cycles a block, beside 4 FMAs a
// lane).  That adder aligns neighbouring products to the largest of them and drops what lies 2^-13 below it: for
// normal values an error of 1.3e-5 of the sum (measured; v_mfma_f32_16x16x32_fp8_fp8 gives the same bits), 300 times
// below bf16's rounding but 100 above fp32's.  fp32 results therefore decode the codes to bf16 (exact) for four
// v_mfma_f32_16x16x32_bf16, which sum as fp32 does (1e-8).
#include "fp8_blocks.h"

#include <type_traits>

namespace {

typedef int int8v __attribute__((ext_vector_type(8)));
typedef int int4v __attribute__((ext_vector_type(4)));

// what a lane reads in place of codes past a row's end, of a row that there is not, and of its scale
__device__ __attribute__((aligned(16))) const uint32_t kZeros[4] = {0, 0, 0, 0};

struct Args {
  const uint8_t* x;
  const float* sx;
  const int32_t* index;  // row of x for each row of y, or null
  const uint8_t* w;
  const float* sw;
  const int32_t* offsets;  // grouped only
  void* y;
  int64_t xs, sxs, xrows, wgs, ws, swgs, sws, ys;
  int64_t rows;   // of y
  int K, N, groups;
  int mt, nt;     // tiles along tokens (grouped: the most there may be) and features
  int out_f32;
  int wide;       // y's rows begin at multiples of 16 bytes
};

// this workgroup's tile: neighbours in the order of tiles run on one XCD (workgroup i runs on XCD i % 8) and
// share its L2; within a band of kBand token tiles the tiles of one feature block follow each other
constexpr int kBand = 8;
__device__ __forceinline__ bool tile_of(const Args& a, int& tm, int& tn) {
  const int64_t total = (int64_t)a.mt * a.nt, per = (total + 7) / 8;
  const int64_t t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || t >= total) return false;
  const int64_t band = t / ((int64_t)kBand * a.nt);
  const int r = static_cast<int>(t - band * kBand * a.nt), high = min(kBand, a.mt - (int)band * kBand);
  tn = r / high;
  tm = (int)band * kBand + r - tn * high;
  return true;
}

// The group and rows of token tile tm: offsets held to [0, rows] and ascending; every wave scans them for itself,
// 64 groups at a time.  False where there are fewer tiles.
template <int BM>
__device__ __forceinline__ bool group_of(const Args& a, int tm, int& group, int64_t& m0, int& count) {
  const int lane = threadIdx.x & 63, rows = static_cast<int>(a.rows);
  int before = 0, least = 0;  // tiles of the groups before, the largest offset so far
  for (int base = 0; base < a.groups; base += 64) {
    const int e = min(base + lane, a.groups - 1);
    int lo = min(max(a.offsets[e], 0), rows), hi = min(max(a.offsets[e + 1], 0), rows);
    lo = max(lo, least);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) lo = max(lo, __shfl_up(lo, o, 64));  // lane 0's own: shfl_up returns it
    hi = max(hi, lo);
    const int tiles = base + lane < a.groups ? (hi - lo + BM - 1) / BM : 0;
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int s = __shfl_up(sum, o, 64);
      if (lane >= o) sum += s;
    }
    const uint64_t past = __ballot(before + sum > tm);
    if (past) {
      const int l = __builtin_ctzll(past);
      group = base + l;
      const int in = tm - before - __builtin_amdgcn_readlane(sum - tiles, l);
      const int r0 = __builtin_amdgcn_readlane(lo, l) + in * BM;
      m0 = r0;
      count = min(BM, __builtin_amdgcn_readlane(hi, l) - r0);
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    least = __builtin_amdgcn_readlane(hi, 63);
  }
  return false;
}

__device__ __forceinline__ void store4(const Args& a, int64_t m, int n, const floatx4_t& v) {
  if (n >= a.N) return;
  if (a.out_f32) {
    float* p = static_cast<float*>(a.y) + m * a.ys + n;
    if (a.wide && n + 4 <= a.N) {
      *reinterpret_cast<floatx4_t*>(p) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) p[i] = v[i];
    }
  } else {
    bf16_t* p = static_cast<bf16_t*>(a.y) + m * a.ys + n;
    if (a.wide && n + 4 <= a.N) {
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) p[i] = f2bf(v[i]);
    }
  }
}

// 16 codes from p, of which n are in the row
__device__ __forceinline__ uint4 codes16(const uint8_t* p, int n) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (n >= 16) {
    __builtin_memcpy(&v, p, 16);  // any alignment
  } else if (n > 0) {
    uint32_t d[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (i < n) d[i >> 2] |= (uint32_t)p[i] << (8 * (i & 3));
    v = make_uint4(d[0], d[1], d[2], d[3]);
  }
  return v;
}

// A lane's 32 codes of one row of a block, and a block's sum of two of them
struct Codes {
  int8v v;
};
struct Decoded {
  bf16x8_t v[4];
};
__device__ __forceinline__ void operand(const int8v& c, Codes& o) { o.v = c; }
__device__ __forceinline__ void operand(const int8v& c, Decoded& o) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[2 * i], 1.0f, false);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[2 * i], 1.0f, true);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[2 * i + 1], 1.0f, false);
    const bf16x2_t e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[2 * i + 1], 1.0f, true);
    o.v[i] = bf16x8_t{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
  }
}
__device__ __forceinline__ floatx4_t block_sum(const Codes& w, const Codes& x) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, floatx4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ floatx4_t block_sum(const Decoded& w, const Decoded& x) {
  floatx4_t p = floatx4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) p = mfma16x16x32(w.v[i], x.v[i], p);
  return p;
}

// A workgroup of WM x WN waves, each TT x FT MFMA tiles of 16 tokens x 16 features; K in chunks of one block.
// The chunk's rows of 128 bytes lie in LDS with their 16-byte pieces exchanged by row (piece p of row r at
// place p ^ key(r)), so that 8 lanes reading one piece of 8 rows hit different banks.  Row i of a wave's MFMA
// tile f is its feature 4 FT (i / 4) + 4 f + i % 4: a lane ends with 4 FT neighbouring features.
template <int WM, int WN, int TT, int FT, bool EXACT, bool GROUPED>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(const Args a) {
  constexpr int BM = 16 * TT * WM, BN = 16 * FT * WN, NW = WM * WN, DI = (BM + BN) / 8 / NW;
  static_assert((BM + BN) % (8 * NW) == 0 && 128 % BN == 0, "tile");
  using Operand = std::conditional_t<EXACT, Decoded, Codes>;
  __shared__ __attribute__((aligned(16))) uint8_t lds[(BM + BN) * 128];
  __shared__ float lsx[BM];
  int tm, tn, group = 0, count;
  int64_t m0;
  if (!tile_of(a, tm, tn)) return;
  if constexpr (GROUPED) {
    if (!group_of<BM>(a, tm, group, m0, count)) return;
  } else {
    m0 = (int64_t)tm * BM;
    count = static_cast<int>(min((int64_t)BM, a.rows - m0));
  }
  const int n0 = tn * BN, lane = threadIdx.x & 63, wv = threadIdx.x >> 6, wm = wv % WM, wn = wv / WM;
  const int li = lane & 15, kg = lane >> 4, nch = (a.K + kFp8Block - 1) / kFp8Block;
  const float* sw = a.sw + group * a.swgs + (n0 / kFp8Block) * a.sws;
  // rows past the tile's are its last one again: their sums are not stored
  auto x_row = [&](int t) -> int64_t {
    const int64_t m = m0 + min(t, count - 1);
    if (!GROUPED || !a.index) return m;
    const int64_t r = a.index[m];
    return r >= 0 && r < a.xrows ? r : -1;
  };
  const uint8_t* src[DI];
  int lim[DI];
#pragma unroll
  for (int j = 0; j < DI; ++j) {
    const int r = (wv * DI + j) * 8 + (lane >> 3), q = r - BM;
    const int key = r < BM ? r & 7 : (q & 3) | (q / (4 * FT) & 1) << 2, at = ((lane & 7) ^ key) * 16;
    const int64_t row = r < BM ? x_row(r) : min(n0 + q, a.N - 1);
    src[j] = (r < BM ? a.x + max(row, (int64_t)0) * a.xs : a.w + group * a.wgs + row * a.ws) + at;
    lim[j] = row < 0 ? 0 : a.K - at;
  }
  const int64_t srow = x_row(min((int)threadIdx.x, BM - 1));
  floatx4_t acc[TT][FT];
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int f = 0; f < FT; ++f) acc[t][f] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  const int piece = (kg ^ (li & 7)) * 16;
  const uint8_t* lx = lds + (wm * TT * 16 + li) * 128;
  const uint8_t* lw = lds + (BM + wn * FT * 16 + (li >> 2) * 4 * FT + (li & 3)) * 128;
  auto frag = [&](const uint8_t* p) {
    const int4v a = *reinterpret_cast<const int4v*>(p + piece), b = *reinterpret_cast<const int4v*>(p + (piece ^ 64));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  for (int c = 0; c < nch; ++c) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < DI; ++j)
      *reinterpret_cast<uint4*>(lds + ((wv * DI + j) * 8) * 128 + lane * 16) =
          codes16(src[j] + c * kFp8Block, lim[j] - c * kFp8Block);
    if (threadIdx.x < BM) lsx[threadIdx.x] = srow < 0 ? 0.f : a.sx[srow * a.sxs + c];
    __syncthreads();
    Operand wf[FT];
#pragma unroll
    for (int f = 0; f < FT; ++f) operand(frag(lw + f * 4 * 128), wf[f]);
    const float s = sw[c];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      Operand xf;
      operand(frag(lx + t * 16 * 128), xf);
      const float st = s * lsx[wm * TT * 16 + t * 16 + li];
#pragma unroll
      for (int f = 0; f < FT; ++f) {
        const floatx4_t p = block_sum(wf[f], xf);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][f][i] = __builtin_fmaf(st, p[i], acc[t][f][i]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    const int m = wm * TT * 16 + t * 16 + li;
    if (m < count) {
#pragma unroll
      for (int f = 0; f < FT; ++f) store4(a, m0 + m, n0 + wn * FT * 16 + kg * 4 * FT + f * 4, acc[t][f]);
    }
  }
}

template <bool GROUPED>
int launch(Args a, hipStream_t st) {
  constexpr int BM = 64, BN = 64;
  const int64_t mt = GROUPED ? (a.rows + min(a.rows, (int64_t)a.groups) * (BM - 1)) / BM : (a.rows + BM - 1) / BM;
  const int64_t nt = (a.N + BN - 1) / BN;
  // a launch has fewer than 2^32 threads
  DSV2_REQUIRE(mt * nt <= 0xfffff8, DSV2_E_SHAPE, "linear_fp8_blocks: %lld rows of %d", (long long)a.rows, a.N);
  a.mt = (int)mt;
  a.nt = (int)nt;
  const dim3 grid((unsigned)((mt * nt + 7) / 8 * 8));
  if (a.out_f32) product_kernel<2, 2, 2, 2, true, GROUPED><<<grid, 256, 0, st>>>(a);
  else product_kernel<2, 2, 2, 2, false, GROUPED><<<grid, 256, 0, st>>>(a);
  return dsv2_launch_status(GROUPED ? "grouped_linear_fp8_blocks" : "linear_fp8_blocks");
}

bool aligned(const void* p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

#define CHECK_PRODUCT(name)                                                                                       \
  DSV2_REQUIRE(out_dtype == DSV2_DTYPE_BF16 || out_dtype == DSV2_DTYPE_F32, DSV2_E_FLAGS, name ": out_dtype %d", \
               out_dtype);                                                                                        \
  DSV2_REQUIRE(rows >= 0 && rows <= 0x7fffffff && K > 0 && K <= 0x7fffff00 && N > 0 && N <= 0x7fffff00, DSV2_E_SHAPE, \
               name ": %lld rows, K %d, N %d", (long long)rows, K, N);                                           \
  if (rows == 0) return DSV2_OK;                                                                                  \
  DSV2_REQUIRE((rows == 1 || y_stride >= N) && x_stride >= 0 && x_scales_stride >= 0 && w_stride >= 0 &&          \
                   w_scales_stride >= 0, DSV2_E_SHAPE, name ": strides");                                         \
  DSV2_REQUIRE(aligned(x_scales, 4) && aligned(w_scales, 4) && aligned(y, out_dtype == DSV2_DTYPE_BF16 ? 2 : 4),  \
               DSV2_E_ALIGN, name ": alignment");

int dsv2_linear_fp8_blocks(const void* x, int64_t x_stride, const float* x_scales, int64_t x_scales_stride, int64_t rows,
                           int K, const void* w, int64_t w_stride, const float* w_scales, int64_t w_scales_stride, int N,
                           void* y, int64_t y_stride, int out_dtype, void* stream) {
  CHECK_PRODUCT("linear_fp8_blocks")
  DSV2_REQUIRE(x && x_scales && w && w_scales && y, DSV2_E_NULL, "linear_fp8_blocks: null pointer");
  const int size = out_dtype == DSV2_DTYPE_BF16 ? 2 : 4;
  Args a{static_cast<const uint8_t*>(x), x_scales, nullptr, static_cast<const uint8_t*>(w), w_scales, nullptr, y,
         x_stride, x_scales_stride, rows, 0, w_stride, 0, w_scales_stride, y_stride, rows, K, N, 1, 0, 0,
         out_dtype == DSV2_DTYPE_F32, dsv2_aligned16(y) && y_stride * size % 16 == 0};
  return launch<false>(a, static_cast<hipStream_t>(stream));
}

int dsv2_grouped_linear_fp8_blocks(const void* x, int64_t x_stride, const float* x_scales, int64_t x_scales_stride,
                                   int64_t x_rows, const int32_t* index, int64_t rows, int K, const void* w,
                                   int64_t w_gstride, int64_t w_stride, const float* w_scales, int64_t w_scales_gstride,
                                   int64_t w_scales_stride, int N, int groups, const int32_t* offsets, void* y,
                                   int64_t y_stride, int out_dtype, void* stream) {
  CHECK_PRODUCT("grouped_linear_fp8_blocks")
  DSV2_REQUIRE(groups > 0 && groups <= 65536 && x_rows >= 0 && (index || x_rows >= rows), DSV2_E_SHAPE,
               "grouped_linear_fp8_blocks: %d groups, %lld rows of x", groups, (long long)x_rows);
  DSV2_REQUIRE(w_gstride >= 0 && w_scales_gstride >= 0, DSV2_E_SHAPE, "grouped_linear_fp8_blocks: strides");
  DSV2_REQUIRE(aligned(offsets, 4) && aligned(index, 4), DSV2_E_ALIGN, "grouped_linear_fp8_blocks: alignment");
  DSV2_REQUIRE((x && x_scales || x_rows == 0) && w && w_scales && offsets && y, DSV2_E_NULL,
               "grouped_linear_fp8_blocks: null pointer");
  const int size = out_dtype == DSV2_DTYPE_BF16 ? 2 : 4;
  Args a{static_cast<const uint8_t*>(x), x_scales, index, static_cast<const uint8_t*>(w), w_scales, offsets, y,
         x_stride, x_scales_stride, x_rows, w_gstride, w_stride, w_scales_gstride, w_scales_stride, y_stride, rows, K, N,
         groups, 0, 0, out_dtype == DSV2_DTYPE_F32, dsv2_aligned16(y) && y_stride * size % 16 == 0};
  return launch<true>(a, static_cast<hipStream_t>(stream));
}
