// Rounding to e4m3 with a fp32 scale for each block of 128 columns: of rows as they are, of weights in
// 128 x 128 blocks, of RMSNorm's output with the residual's addition before it, of SwiGLU's output.
// No counterpart in the reference, whose path is bf16 throughout.
//
// A block of a row is 16 lanes of 8 values: one 16-byte load a lane of bf16, the largest value by four
// DPP steps, one 8-byte store of codes.  All of it is bound by memory (2 to 9 bytes a value for some 10
// to 30 instructions), for few rows by the launch and one trip to memory.  MI355X, bf16, a call in a replayed graph over
// three sets of tensors: 64 x 2,048 2.2 us, an empty launch 1.7; SwiGLU of 49,152 x 1,408 58 to 61 us, 5.7 to 6.0 TB/s (a
// large copy 5.7: some of it stays in the last-level cache); 384 x 1,408 2.9.
#include "fp8_blocks.h"

namespace {

template <bool NT>
__device__ __forceinline__ uint4 load16(const void* p) {
  if constexpr (NT) return ldg16_nt(p);
  else return ldg16(p);
}
__device__ __forceinline__ uint4 load16_any(const void* p) {  // of any alignment
  uint4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}

__device__ __forceinline__ void floats(const uint4& a, const uint4& b, float (&f)[8]) {
  f[0] = __uint_as_float(a.x), f[1] = __uint_as_float(a.y), f[2] = __uint_as_float(a.z), f[3] = __uint_as_float(a.w);
  f[4] = __uint_as_float(b.x), f[5] = __uint_as_float(b.y), f[6] = __uint_as_float(b.z), f[7] = __uint_as_float(b.w);
}

// a lane's 8 values from p, of which n are in the row.  VEC: all or none, at multiples of 16 bytes; else all of them by
// the same loads at any alignment (a lane's bytes then lie in two lines now and then), a row's last few one by one
template <typename T, bool VEC, bool NT = false>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, float (&f)[8]) {
  if constexpr (VEC) {
    const uint4 z = make_uint4(0, 0, 0, 0);
    if constexpr (sizeof(T) == 2) {
      unpack8(n > 0 ? load16<NT>(p) : z, f);
    } else {
      const uint4 a = n > 0 ? load16<NT>(p) : z, b = n > 0 ? load16<NT>(p + 4) : z;
      floats(a, b, f);
    }
  } else if (n >= 8) {
    if constexpr (sizeof(T) == 2) unpack8(load16_any(p), f);
    else floats(load16_any(p), load16_any(p + 4), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = 0.f;
      if (i < n) {
        if constexpr (sizeof(T) == 2) f[i] = bf2f(p[i]);
        else f[i] = p[i];
      }
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, const float (&f)[8]) {
  if (VEC ? n > 0 : n >= 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 v = pack8(f);
      if constexpr (VEC) *reinterpret_cast<uint4*>(p) = v;
      else __builtin_memcpy(p, &v, 16);
    } else {
      if constexpr (VEC) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        __builtin_memcpy(p, f, 32);
      }
    }
  } else if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 2) p[i] = f2bf(f[i]);
        else p[i] = f[i];
      }
  }
}

template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* __restrict__ p, int n, const Fp8Rounding& q, const float (&f)[8]) {
  const uint2 v = make_uint2(fp8x4(q(f[0]), q(f[1]), q(f[2]), q(f[3])), fp8x4(q(f[4]), q(f[5]), q(f[6]), q(f[7])));
  if (VEC ? n > 0 : n >= 8) {
    if constexpr (VEC) *reinterpret_cast<uint2*>(p) = v;
    else __builtin_memcpy(p, &v, 8);
  } else if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = static_cast<uint8_t>((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ uint32_t max8(const float (&f)[8]) {
  uint32_t m = abs_bits(f[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max(m, abs_bits(f[i]));
  return m;
}

// ---------------------------------------------------------------------------
// Rows, and SwiGLU: every block for itself, 16 lanes a block.
// ---------------------------------------------------------------------------
struct BlockArgs {
  const void* x;      // gate for SwiGLU
  const void* up;
  int64_t x_stride, up_stride;
  int64_t n_blocks;   // rows * blocks of a row
  int K, kb;          // columns, blocks of a row
  uint8_t* codes;     // [rows, K]
  float* scales;      // [rows, kb]
};

// silu(g) u = g u / (1 + exp(-g)) in fp32.  exp(-g) = 2^-(t + r), t the rounded product g log2(e) and r what its
// rounding lost: v_exp_f32 of t alone is off by |t| / 2 ulp.  The quotient g / d by v_rcp_f32 with one residual of its own,
// rounded once (the product with a rounded 1 / d is rounded twice: 0.94 half steps rms in the end for 0.84).
__device__ __forceinline__ float swiglu(float g, float u) {
  constexpr float l2e = 1.44269504088896f, l2e_lo = 1.92596299e-8f, ln2 = 0.693147180559945f;
  // a gate past 2.3e38 takes t out of range and r to -inf, which times exp2(-t) = 0 would be NaN; where the exponential
  // counts r is within 2^-15
  const float t = g * l2e, lost = __builtin_fmaf(g, l2e_lo, __builtin_fmaf(g, l2e, -t)), r = __builtin_fmaxf(lost, -1.f) * ln2;
  if (t < -120.f) {
    // 1 + exp(-g) = exp(-g) in fp32, and soon past its range: 2^130 exp(g) instead, a normal number as long as the largest
    // u brings the product to a code; u takes half of the factor back before the product, which has to stay in range
    if (t < -300.f && g > -__builtin_inff()) return 0.f * g * u;
    const float e = __builtin_amdgcn_exp2f(t + 130.f);
    return g * __builtin_fmaf(r, e, e) * (u * 0x1p-64f) * 0x1p-66f;
  }
  const float e = __builtin_amdgcn_exp2f(-t), d = 1.f + __builtin_fmaf(-r, e, e);
  const float ri = __builtin_amdgcn_rcpf(d), q = g * ri;
  return __builtin_fmaf(__builtin_fmaf(-q, d, g), ri, q) * u;
}

// NB blocks for each 16 lanes, 16 NB a workgroup
template <typename T, bool SILU, bool VEC, int NB, bool NT>
__global__ __launch_bounds__(256) void block_kernel(const BlockArgs a) {
  const int64_t b0 = blockIdx.x * (int64_t)(16 * NB), row0 = b0 / a.kb;
  const T* const x = reinterpret_cast<const T*>(a.x);
  float f[NB][8], u[SILU ? NB : 1][8];
  int64_t row[NB];
  int c[NB];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const uint32_t at = static_cast<uint32_t>(b0 - row0 * a.kb) + (threadIdx.x >> 4) + 16 * i, down = at / (uint32_t)a.kb;
    row[i] = row0 + down;
    c[i] = static_cast<int>(at - down * a.kb) * kFp8Block + (threadIdx.x & 15) * 8;
    const int n = b0 + (threadIdx.x >> 4) + 16 * i < a.n_blocks ? a.K - c[i] : 0;
    load8<T, VEC, NT>(x + row[i] * a.x_stride + c[i], n, f[i]);
    if constexpr (SILU) load8<T, VEC, NT>(reinterpret_cast<const T*>(a.up) + row[i] * a.up_stride + c[i], n, u[i]);
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const int64_t b = b0 + (threadIdx.x >> 4) + 16 * i;
    if (b >= a.n_blocks) return;  // whole 16-lane rows leave: the DPP steps stay within one
    if constexpr (SILU) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[i][j] = swiglu(f[i][j], u[i][j]);
    }
    const uint32_t m = max(row_max(max8(f[i])), kLeastBits);
    store_codes<VEC>(a.codes + row[i] * a.K + c[i], a.K - c[i], Fp8Rounding(m), f[i]);
    if ((threadIdx.x & 15) == 0) a.scales[b] = fp8_scale(m);
  }
}

// ---------------------------------------------------------------------------
// Weights: one workgroup a 128 x 128 block, its values in registers between the maximum and the codes, so that memory
// is read once (MI355X: 21,888 x 2,048 bf16 25.3 us, 5.3 TB/s).
// ---------------------------------------------------------------------------
struct WeightArgs {
  const void* x;
  int64_t x_stride, x_gstride;
  int64_t rows;  // of a matrix
  int K, kb, rb;  // columns; blocks of a row, of a column
  uint8_t* codes;
  float* scales;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void weight_kernel(const WeightArgs a) {
  __shared__ uint32_t red[4];
  const uint32_t per = (uint32_t)a.rb * a.kb, at = blockIdx.x % per, down = at / a.kb;
  const int64_t g = blockIdx.x / per, r0 = (int64_t)down * kFp8Block;
  const int c = static_cast<int>(at - down * a.kb) * kFp8Block + (threadIdx.x & 15) * 8;
  const T* x = reinterpret_cast<const T*>(a.x) + g * a.x_gstride + c;
  float f[8][8];
  uint32_t m = kLeastBits;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + 16 * i + (threadIdx.x >> 4);
    load8<T, VEC>(x + min(r, a.rows - 1) * a.x_stride, r < a.rows ? a.K - c : 0, f[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, max8(f[i]));
  m = row_max(m);
#pragma unroll
  for (int i = 16; i < 64; i += 16) m = max(m, static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(m), i)));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(red[0], red[1]), max(red[2], red[3]));
  const Fp8Rounding q(m);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = r0 + 16 * i + (threadIdx.x >> 4);
    if (r < a.rows) store_codes<VEC>(a.codes + (g * a.rows + r) * a.K + c, a.K - c, q, f[i]);
  }
  if (threadIdx.x == 0) a.scales[blockIdx.x] = fp8_scale(m);
}

// ---------------------------------------------------------------------------
// RMSNorm: h = x + residual, y = h w / sqrt(mean(h^2) + eps).  The row's factor cancels from 448 y / max |y|, so the
// codes are those of h w (exact products for bf16), need no sum and leave in the same pass; the scales wait
// for it.  WPR waves a row; its blocks' maxima stay in registers where NCH chunks of 512 columns a wave
// hold it, else (NCH = 0) the scales are stored without the factor and read back by the lanes that wrote them.
// ---------------------------------------------------------------------------
struct NormArgs {
  const void *x, *residual, *weight;
  int64_t x_stride, res_stride, rows;
  int K, kb;
  float eps;
  uint8_t* codes;
  float* scales;
  void* sum;  // [rows, K]: h, with a residual
};

template <typename T, bool RES, bool VEC>
__device__ __forceinline__ uint32_t norm_chunk(const NormArgs& a, int64_t row, int c, float& ss) {
  const int n = a.K - c;
  float h[8], w[8];
  load8<T, VEC>(reinterpret_cast<const T*>(a.x) + row * a.x_stride + c, n, h);
  load8<T, VEC>(reinterpret_cast<const T*>(a.weight) + c, n, w);
  if constexpr (RES) {
    float r[8];
    load8<T, VEC>(reinterpret_cast<const T*>(a.residual) + row * a.res_stride + c, n, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[i] += r[i];
      if constexpr (sizeof(T) == 2) h[i] = rbf(h[i]);  // the sum as it is stored and read by the next layer
    }
    store8<T, VEC>(reinterpret_cast<T*>(a.sum) + row * a.K + c, n, h);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    ss = __builtin_fmaf(h[i], h[i], ss);
    h[i] *= w[i];
  }
  const uint32_t m = max(row_max(max8(h)), kLeastBits);
  store_codes<VEC>(a.codes + row * a.K + c, n, Fp8Rounding(m), h);
  return m;
}

template <typename T, int WPR, int NCH, bool RES, bool VEC>
__global__ __launch_bounds__(256) void norm_kernel(const NormArgs a) {
  __shared__ float red[4];
  const int wv = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = WPR == 4 ? blockIdx.x : blockIdx.x * (int64_t)4 + wv;
  if (row >= a.rows) return;  // WPR == 4: never; else no barrier follows
  const int first = (WPR == 4 ? wv * 512 : 0) + lane * 8;
  constexpr int step = WPR * 512;
  float* scales = a.scales + row * a.kb;
  const bool lead = (lane & 15) == 0;
  float ss = 0.f;
  uint32_t m[NCH ? NCH : 1];
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) m[i] = norm_chunk<T, RES, VEC>(a, row, first + i * step, ss);
  } else {
    for (int c = first; c - lane * 8 < a.K; c += step) {
      const uint32_t mm = norm_chunk<T, RES, VEC>(a, row, c, ss);
      if (lead && c < a.K) scales[c / kFp8Block] = fp8_scale(mm);
    }
  }
  ss = wave_sum(ss);
  if constexpr (WPR == 4) {
    if (lane == 0) red[wv] = ss;
    __syncthreads();
    ss = (red[0] + red[1]) + (red[2] + red[3]);
  }
  const float rstd = rsqrtf(ss / a.K + a.eps);
  if (!lead) return;
  if constexpr (NCH > 0) {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int c = first + i * step;
      if (c < a.K) scales[c / kFp8Block] = fp8_scale(m[i]) * rstd;
    }
  } else {
    for (int c = first; c < a.K; c += step) scales[c / kFp8Block] *= rstd;
  }
}

// A wave a row where it holds the row in one chunk, else four (MI355X, bf16 with a residual, a wave / four: 8,192 x
// 512 7.4 / 9.1 us, 65,536 x 128 21 / 45; in four chunks 8,192 x 2,048 19.3 / 18.8, 64 x 2,048 4.1 / 2.7).  Maxima in
// registers or scales read back: 64 x 2,048 2.7 / 3.1, 64 x 4,096 3.2 / 3.5, 64 x 8,192 4.3 / 4.9, 4,096 x 8,192
// 38.8 / 39.4.  8,192 x 2,048 moves 118 MB in 18.6 to 21.8 us, 5.4 to 6.3 TB/s (a copy past the caches 5.7: some of it
// stays in them).
template <typename T, bool RES, bool VEC>
void launch_norm(const NormArgs& a, hipStream_t st) {
  if (a.K <= 512) {
    norm_kernel<T, 1, 1, RES, VEC><<<dim3((unsigned)((a.rows + 3) / 4)), 256, 0, st>>>(a);
  } else if (a.K <= 2048) {
    norm_kernel<T, 4, 1, RES, VEC><<<dim3((unsigned)a.rows), 256, 0, st>>>(a);
  } else if (a.K <= 4096) {
    norm_kernel<T, 4, 2, RES, VEC><<<dim3((unsigned)a.rows), 256, 0, st>>>(a);
  } else if (a.K <= 8192) {
    norm_kernel<T, 4, 4, RES, VEC><<<dim3((unsigned)a.rows), 256, 0, st>>>(a);
  } else {
    norm_kernel<T, 4, 0, RES, VEC><<<dim3((unsigned)a.rows), 256, 0, st>>>(a);
  }
}

template <typename T>
void launch_norm(const NormArgs& a, bool vec, hipStream_t st) {
  if (a.residual) {
    if (vec) launch_norm<T, true, true>(a, st);
    else launch_norm<T, true, false>(a, st);
  } else {
    if (vec) launch_norm<T, false, true>(a, st);
    else launch_norm<T, false, false>(a, st);
  }
}

template <typename T, bool SILU, int NB, bool NT>
void launch_blocks(const BlockArgs& a, bool vec, hipStream_t st) {
  const dim3 grid((unsigned)((a.n_blocks + 16 * NB - 1) / (16 * NB)));
  if (vec) block_kernel<T, SILU, true, NB, NT><<<grid, 256, 0, st>>>(a);
  else block_kernel<T, SILU, false, NB, false><<<grid, 256, 0, st>>>(a);
}

// One block for each 16 lanes, two where there are many workgroups either way (MI355X, calls in a replayed graph over
// three sets of tensors, one / two: 16,384 blocks of rows 3.1 / 3.2 us, 65,536 6.6 / 6.5, 131,072 10.9 / 10.4, 640,000
// 47 / 41), but not of SwiGLU, which hides its loads by its own instructions (33,000 blocks 6.9 / 7.7; at
// 330,000 the two are even, 41.3 / 39.9 and over one set 35.4 / 35.1).  Two with non-temporal loads for what cannot stay in
// the 256 MB of the last-level cache (80,000 x 2,048 rows 85.5 -> 77.3; 49,152 x 1,408 SwiGLU 63.9 -> 60.0; in the
// cache, 8,192 rows 10.3 -> 11.5, 30,000 of SwiGLU over one set 35.1 -> 40.7).
template <typename T, bool SILU>
void launch_blocks(const BlockArgs& a, bool vec, hipStream_t st) {
  const int64_t bytes = a.n_blocks * kFp8Block * (int64_t)sizeof(T) * (SILU ? 2 : 1);
  if (bytes > 256ll << 20) launch_blocks<T, SILU, 2, true>(a, vec, st);
  else if (!SILU && a.n_blocks > 98304) launch_blocks<T, false, 2, false>(a, vec, st);
  else launch_blocks<T, SILU, 1, false>(a, vec, st);
}

// rows that a kernel's 16-byte loads may take: whole groups of 8 values at multiples of 16 bytes
bool wide(const void* p, int64_t stride, int64_t rows, int size) {
  return dsv2_aligned16(p) && (rows <= 1 || stride * size % 16 == 0);
}

constexpr int64_t kMaxGrid = 0xffffff;  // workgroups of 256: a launch has fewer than 2^32 threads

// pointers and strides of rows of values of `size` bytes
bool fits(const void* p, int64_t stride, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0 && stride >= 0; }

}  // namespace

#define CHECK_COMMON(name)                                                                                      \
  DSV2_REQUIRE(dtype == DSV2_DTYPE_BF16 || dtype == DSV2_DTYPE_F32, DSV2_E_FLAGS, name ": dtype %d", dtype);    \
  DSV2_REQUIRE(rows >= 0 && K > 0 && K <= 1 << 30, DSV2_E_SHAPE, name ": %lld rows of %d", (long long)rows, K); \
  if (rows == 0) return DSV2_OK;

int dsv2_quantize_fp8_blocks(const void* x, int64_t x_stride, int64_t x_gstride, int64_t groups, int64_t rows, int K,
                             int dtype, int block_rows, void* codes, float* scales, void* stream) {
  CHECK_COMMON("quantize_fp8_blocks")
  DSV2_REQUIRE(block_rows == 1 || block_rows == kFp8Block, DSV2_E_FLAGS, "quantize_fp8_blocks: blocks of %d rows",
               block_rows);
  DSV2_REQUIRE(groups >= 0 && (block_rows > 1 || groups == 1), DSV2_E_SHAPE, "quantize_fp8_blocks: %lld groups",
               (long long)groups);
  if (groups == 0) return DSV2_OK;
  DSV2_REQUIRE(x && codes && scales, DSV2_E_NULL, "quantize_fp8_blocks: null pointer");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int size = dtype == DSV2_DTYPE_BF16 ? 2 : 4;
  DSV2_REQUIRE(fits(x, x_stride, size) && fits(scales, x_gstride, 4), DSV2_E_ALIGN, "quantize_fp8_blocks: alignment");
  const int kb = (K + kFp8Block - 1) / kFp8Block;
  const bool vec = K % 8 == 0 && wide(x, x_stride, rows, size) && wide(x, x_gstride, groups, size) &&
                   (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
  if (block_rows == 1) {
    DSV2_REQUIRE(rows <= (kMaxGrid * 16 - 15) / kb, DSV2_E_SHAPE, "quantize_fp8_blocks: %lld rows", (long long)rows);
    const BlockArgs a{x, nullptr, x_stride, 0, rows * kb, K, kb, static_cast<uint8_t*>(codes), scales};
    if (dtype == DSV2_DTYPE_BF16) launch_blocks<bf16_t, false>(a, vec, st);
    else launch_blocks<float, false>(a, vec, st);
  } else {
    const int64_t rb = (rows + kFp8Block - 1) / kFp8Block;
    DSV2_REQUIRE(rb <= kMaxGrid / kb && rb * kb <= kMaxGrid / groups, DSV2_E_SHAPE,
                 "quantize_fp8_blocks: %lld matrices of %lld rows", (long long)groups, (long long)rows);
    const WeightArgs a{x, x_stride, x_gstride, rows, K, kb, (int)rb, static_cast<uint8_t*>(codes), scales};
    const dim3 grid((unsigned)(groups * rb * kb));
    if (dtype == DSV2_DTYPE_BF16) {
      if (vec) weight_kernel<bf16_t, true><<<grid, 256, 0, st>>>(a);
      else weight_kernel<bf16_t, false><<<grid, 256, 0, st>>>(a);
    } else {
      if (vec) weight_kernel<float, true><<<grid, 256, 0, st>>>(a);
      else weight_kernel<float, false><<<grid, 256, 0, st>>>(a);
    }
  }
  return dsv2_launch_status("quantize_fp8_blocks");
}

int dsv2_rmsnorm_fp8_blocks(const void* x, int64_t x_stride, const void* residual, int64_t res_stride,
                            const void* weight, float eps, int64_t rows, int K, int dtype, void* codes, float* scales,
                            void* sum, void* stream) {
  CHECK_COMMON("rmsnorm_fp8_blocks")
  DSV2_REQUIRE(rows <= kMaxGrid, DSV2_E_SHAPE, "rmsnorm_fp8_blocks: %lld rows", (long long)rows);
  DSV2_REQUIRE(x && weight && codes && scales && (!residual || sum), DSV2_E_NULL, "rmsnorm_fp8_blocks: null pointer");
  const int size = dtype == DSV2_DTYPE_BF16 ? 2 : 4, kb = (K + kFp8Block - 1) / kFp8Block;
  DSV2_REQUIRE(fits(x, x_stride, size) && fits(residual, res_stride, size) && fits(weight, 0, size) &&
                   fits(sum, 0, size) && fits(scales, 0, 4), DSV2_E_ALIGN, "rmsnorm_fp8_blocks: alignment");
  const bool vec = K % 8 == 0 && wide(x, x_stride, rows, size) && (!residual || wide(residual, res_stride, rows, size)) &&
                   dsv2_aligned16(weight) && (!residual || dsv2_aligned16(sum)) &&
                   (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
  const NormArgs a{x, residual, weight, x_stride, res_stride, rows, K, kb, eps, static_cast<uint8_t*>(codes), scales,
                   sum};
  if (dtype == DSV2_DTYPE_BF16) launch_norm<bf16_t>(a, vec, static_cast<hipStream_t>(stream));
  else launch_norm<float>(a, vec, static_cast<hipStream_t>(stream));
  return dsv2_launch_status("rmsnorm_fp8_blocks");
}

int dsv2_silu_mul_fp8_blocks(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, int64_t rows,
                             int K, int dtype, void* codes, float* scales, void* stream) {
  CHECK_COMMON("silu_mul_fp8_blocks")
  DSV2_REQUIRE(gate && up && codes && scales, DSV2_E_NULL, "silu_mul_fp8_blocks: null pointer");
  const int size = dtype == DSV2_DTYPE_BF16 ? 2 : 4, kb = (K + kFp8Block - 1) / kFp8Block;
  DSV2_REQUIRE(rows <= (kMaxGrid * 16 - 15) / kb, DSV2_E_SHAPE, "silu_mul_fp8_blocks: %lld rows", (long long)rows);
  DSV2_REQUIRE(fits(gate, gate_stride, size) && fits(up, up_stride, size) && fits(scales, 0, 4), DSV2_E_ALIGN,
               "silu_mul_fp8_blocks: alignment");
  const bool vec = K % 8 == 0 && wide(gate, gate_stride, rows, size) && wide(up, up_stride, rows, size) &&
                   (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
  const BlockArgs a{gate, up, gate_stride, up_stride, rows * kb, K, kb, static_cast<uint8_t*>(codes), scales};
  if (dtype == DSV2_DTYPE_BF16) launch_blocks<bf16_t, true>(a, vec, static_cast<hipStream_t>(stream));
  else launch_blocks<float, true>(a, vec, static_cast<hipStream_t>(stream));
  return dsv2_launch_status("silu_mul_fp8_blocks");
}
