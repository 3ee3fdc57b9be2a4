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
// lane).  That adder aligns the products of 8 neighbouring columns to the largest of them and drops what lies 2^-13 below
// it: for normal values an error of 1.3e-5 of the sum (measured; v_mfma_f32_16x16x32_fp8_fp8 gives the same bits), 300
// times below bf16's rounding but 100 above fp32's.  Beside 448 * 448 and its negative a product of 2^3 is kept and one of
// 2^2 lost in the same 8 columns, 2^-8 kept and 2^-9 lost in the next 8, and none behind them.  fp32 results
// decode the codes to bf16 (exact) for four v_mfma_f32_16x16x32_bf16, which sum as fp32 does (1e-8).
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

// Tile t in the order that shares most: within a band of kBand token tiles the tiles of one feature block follow
// each other.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_at(uint32_t t, int mt, int nt, int& tm, int& tn) {
  const uint32_t band = t / ((uint32_t)kBand * nt), r = t - band * kBand * nt;
  const uint32_t high = min((uint32_t)kBand, mt - band * kBand);
  tn = r / high;
  tm = band * kBand + r - tn * high;
}

// Up to 64 groups' rows and token tiles, a group a lane.  Offsets are held to [0, rows] and ascending.
struct Groups {
  int lo, hi;  // rows lo .. hi - 1
  int tiles;   // of this group and those before it in the 64
};
template <int BM>
__device__ __forceinline__ Groups scan_groups(const Args& a, int base, int least) {
  const int lane = threadIdx.x & 63, rows = static_cast<int>(a.rows), e = min(base + lane, a.groups - 1);
  Groups g;
  g.lo = max(min(max(a.offsets[e], 0), rows), least);
  const int end = min(max(a.offsets[e + 1], 0), rows);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) g.lo = max(g.lo, __shfl_up(g.lo, o, 64));  // the lowest lanes: their own
  g.hi = max(end, g.lo);
  g.tiles = base + lane < a.groups ? (g.hi - g.lo + BM - 1) / BM : 0;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int s = __shfl_up(g.tiles, o, 64);
    if (lane >= o) g.tiles += s;
  }
  return g;
}

// the group and rows of the 64 groups' token tile tm, if it is one of theirs
template <int BM>
__device__ __forceinline__ bool find_tile(const Groups& g, int tm, int& l, int64_t& m0, int& count) {
  const uint64_t past = __ballot(g.tiles > tm);
  if (!past) return false;
  l = __builtin_ctzll(past);
  const int before = l ? __builtin_amdgcn_readlane(g.tiles, l - 1) : 0;
  const int r0 = __builtin_amdgcn_readlane(g.lo, l) + (tm - before) * BM;
  m0 = r0;
  count = min(BM, __builtin_amdgcn_readlane(g.hi, l) - r0);
  return true;
}

// all groups' token tiles; `last`: what the last 64 (up to 64: all) groups are
template <int BM>
__device__ __forceinline__ int all_tiles(const Args& a, Groups& last) {
  int sum = 0, least = 0;
  for (int base = 0; base < a.groups; base += 64) {
    last = scan_groups<BM>(a, base, least);
    sum += __builtin_amdgcn_readlane(last.tiles, 63);
    least = __builtin_amdgcn_readlane(last.hi, 63);
  }
  return sum;
}

// token tile tm of all groups (there is one); `all`: the groups, where they are up to 64
template <int BM>
__device__ __forceinline__ void group_of(const Args& a, const Groups& all, int tm, int& group, int64_t& m0, int& count) {
  if (a.groups <= 64) {
    find_tile<BM>(all, tm, group, m0, count);
    return;
  }
  int least = 0;
  for (int base = 0; base < a.groups; base += 64) {
    const Groups g = scan_groups<BM>(a, base, least);
    if (find_tile<BM>(g, tm, group, m0, count)) {
      group += base;
      return;
    }
    tm -= __builtin_amdgcn_readlane(g.tiles, 63);
    least = __builtin_amdgcn_readlane(g.hi, 63);
  }
}

// This workgroup's tile, if it has one: neighbours in tile_at's order run on one XCD (workgroup i runs on XCD
// i % 8) and share its L2.
template <int BM, bool GROUPED>
__device__ __forceinline__ bool tile_of(const Args& a, int& tn, int& group, int64_t& m0, int& count) {
  Groups all;
  const int mt = GROUPED ? all_tiles<BM>(a, all) : a.mt;
  const uint32_t total = (uint32_t)mt * a.nt, per = (total + 7) / 8;
  const uint32_t t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || t >= total) return false;
  int tm;
  tile_at(t, mt, a.nt, tm, tn);
  if constexpr (GROUPED) {
    group_of<BM>(a, all, tm, group, m0, count);
  } else {
    m0 = (int64_t)tm * BM;
    count = static_cast<int>(min((int64_t)BM, a.rows - m0));
  }
  return true;
}

// features n .. n + 3 of row m; rows may begin at any multiple of a value
__device__ __forceinline__ void store4(const Args& a, int64_t m, int n, const floatx4_t& v) {
  if (a.out_f32) {
    float* const p = static_cast<float*>(a.y) + m * a.ys + n;
    if (n + 4 <= a.N) {
      __builtin_memcpy(p, &v, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (n + i < a.N) p[i] = v[i];
    }
  } else {
    bf16_t* const p = static_cast<bf16_t*>(a.y) + m * a.ys + n;
    const uint2 w = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
    if (n + 4 <= a.N) {
      __builtin_memcpy(p, &w, 8);
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (n + i < a.N) p[i] = static_cast<bf16_t>((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
    }
  }
}

// features n .. n + 7 of a row of N, at any alignment
__device__ __forceinline__ void store8_any(bf16_t* row, int n, int N, const u32x4_t& v) {
  if (n + 8 <= N) {
    __builtin_memcpy(row + n, &v, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (n + i < N) row[n + i] = static_cast<bf16_t>(v[i >> 1] >> (16 * (i & 1)));
  }
}

// 16 codes from p, at any alignment, of which n are in the row
__device__ __forceinline__ uint4 codes16(const uint8_t* p, int n) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (n >= 16) {
    __builtin_memcpy(&v, p, 16);
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

// ---------------------------------------------------------------------------
// A tile by KW groups of WM x WN waves, each wave TT x FT MFMA tiles of 16 tokens x 16 features; group i takes every
// KW-th block of K from block i on.  A block's rows of 128 bytes lie in LDS with their 16-byte pieces exchanged
// by row (piece p of row r at place p ^ key(r)), so that 8 lanes reading one piece of 8 rows hit different banks.  Row
// i of a wave's MFMA tile f is its feature 4 FT (i / 4) + 4 f + i % 4: a lane ends with 4 FT neighbouring features.
//
// Rows of whole 16 codes at multiples of 16 bytes (ANY false) are streamed into LDS without registers
// (global_load_lds): each group has a ring of ST stages, ST - 1 of them requested ahead, and a block's scales come the
// same way, 64 a load.  Other rows go through registers, one block ahead of two stages.  A group of one wave needs no
// barrier: its own waits order its loads and reads.  At the end the groups' sums meet in LDS, in fixed order.
//
// Few rows over a long K load 50 to 55 bytes a ns and CU on MI355X whatever the depth of the ring (2 to 8), the waves or
// the tile: 64 x 2,048 x 10,944 takes 11.3 us, 9.5 of them for 525 KB a CU.  What holds them there is not known, but not
// the CU's load rate: 128 x 128 tiles load 68, and loads alone reach 150 from L2 (80 where rows straddle lines, which
// costs a twentieth here: rows 11,008 apart take 11.0).  Half the bytes a CU gain a tenth.  Tiles are small enough for
// 256 CUs first, and large only beyond (1 x 3,648 x 2,048 3.6 us, 1.7 of them an empty launch; 1,024 x 2,816 x 2,048 17).
// ---------------------------------------------------------------------------
// 16 (4) bytes a lane from src to LDS, lane after lane from dst; in functions of their own: with the builtin in a
// template hipcc drops the kernel's host launch stub
__device__ __forceinline__ void load_lds16(const void* src, uint8_t* dst) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}
// with the non-temporal hint: bytes that nothing reads again soon
__device__ __forceinline__ void load_lds16_nt(const void* src, uint8_t* dst) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 16, 0, 2);
}
__device__ __forceinline__ void load_lds4(const void* src, uint8_t* dst) {
  __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 4, 0, 0);
}

// 16 bytes a lane at base + voffset + soffset to LDS; zeros where voffset is past the resource's size
__device__ __forceinline__ void buffer_lds16(__amdgpu_buffer_rsrc_t base, uint8_t* dst, int voffset, int soffset) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(base, (__attribute__((address_space(3))) void*)dst, 16, voffset, soffset, 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(bytes), 0x00020000);
}

template <int WM, int WN, int TT, int FT, int KW, int ST>
struct Ring {
  static constexpr int BM = 16 * TT * WM, BN = 16 * FT * WN, NW = WM * WN;
  static constexpr int DI = (BM + BN) / 8 / NW;               // loads of codes a wave and stage
  static constexpr int NB = BN > 128 ? BN / 128 : 1;           // scales of features
  static constexpr int XS = (BM + NB + 63) / 64;               // loads of scales: the tokens', then the features'
  static constexpr int SI = (XS + NW - 1) / NW;                // loads of scales a wave and stage
  static constexpr int kCodes = (BM + BN) * 128, kStage = kCodes + SI * NW * 256;
  static constexpr int kRing = KW * ST * kStage;
  static constexpr int kLds = KW > 1 && KW * NW * TT * FT * 1024 > kRing ? KW * NW * TT * FT * 1024 : kRing;
  static constexpr int kThreads = 64 * NW * KW;
  static_assert((BM + BN) % (8 * NW) == 0 && BM % 8 == 0 && kLds <= 160 * 1024, "tile");
  static_assert(BN <= 128 ? 128 % BN == 0 : BN % 128 == 0, "a tile's features are whole blocks or in one");
  static_assert(ST >= 2 && (ST - 2) * (DI + SI) < 64, "vmcnt counts to 63");
};

template <int WM, int WN, int TT, int FT, int KW, int ST, bool NT, bool ANY, bool EXACT, bool GROUPED>
__global__ __launch_bounds__(64 * WM * WN * KW) void ring_kernel(const Args a) {
  using R = Ring<WM, WN, TT, FT, KW, ST>;
  using Operand = std::conditional_t<EXACT, Decoded, Codes>;
  static_assert(!NT || WM * WN == 1, "a load is of tokens or of features");
  static_assert(!ANY || ST == 2, "one block in registers");
  constexpr int BM = R::BM, BN = R::BN, NW = R::NW, DI = R::DI, SI = R::SI;
  // With many matrix instructions a block its fragments are read before the next loads are issued, which holds a wave
  // back, and sums are added two instructions behind (MI355X: 1,024 x 2,816 x 2,048 17.6 -> 16.9 us, 2,048 x 2,816 x 2,048
  // 25.0 -> 23.9, 128 x 64 tiles 47 -> 44).  With few of them the loads' way is the longer one and they go first (32 x
  // 32 tiles at 128 x 2,048 x 10,944 16.1 us, behind the fragments 18.5), as do those through registers to bf16 results.
  constexpr bool kLate = TT * FT >= 8 && (EXACT || !ANY);
  extern __shared__ __attribute__((aligned(16))) uint8_t ring[];
  int tn, group = 0, count = 0;  // no rows, should the offsets change between two looks at them
  int64_t m0 = 0;
  if (!tile_of<BM, GROUPED>(a, tn, group, m0, count)) return;
  const int n0 = tn * BN, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kw = wave / NW, wv = wave % NW, wm = wv % WM, wn = wv / WM;
  const int li = lane & 15, kg = lane >> 4, nch = (a.K + kFp8Block - 1) / kFp8Block;
  // the row of x behind row t of the tile; -1: none, and zeros are read for it
  auto x_row = [&](int t) -> int64_t {
    if (t >= count) return -1;
    if (!GROUPED || !a.index) return m0 + t;
    const int64_t r = a.index[m0 + t];
    return r >= 0 && r < a.xrows ? r : -1;
  };
  const uint8_t* zeros = reinterpret_cast<const uint8_t*>(kZeros);
  const uint8_t* src[DI];
  int lim[DI];  // codes of the row from src on
#pragma unroll
  for (int j = 0; j < DI; ++j) {
    const int r = (wv * DI + j) * 8 + (lane >> 3), q = r - BM;
    const int key = r < BM ? r & 7 : (q & 3) | (q / (4 * FT) & 1) << 2, at = ((lane & 7) ^ key) * 16;
    const int64_t row = r < BM ? x_row(r) : min(n0 + q, a.N - 1);
    src[j] = (r < BM ? a.x + row * a.xs : a.w + group * a.wgs + row * a.ws) + at;
    lim[j] = row < 0 ? 0 : a.K - at;
  }
  const float* ssrc[SI];
#pragma unroll
  for (int j = 0; j < SI; ++j) {
    const int i = (wv + NW * j) * 64 + lane;  // one more scale a lane than needed costs a line of memory each
    ssrc[j] = nullptr;
    if (i < BM) {
      const int64_t row = x_row(i);
      if (row >= 0) ssrc[j] = a.sx + row * a.sxs;
    } else if (i < BM + R::NB) {
      ssrc[j] = a.sw + group * a.swgs + min(n0 / kFp8Block + i - BM, (a.N - 1) / kFp8Block) * a.sws;
    }
  }
  uint8_t* const mine = ring + kw * ST * R::kStage;
  uint4 held[ANY ? DI : 1];
  float factors[ANY ? SI : 1];
  // block c to the stage, or (ANY) into registers and from there to the stage
  auto issue = [&](int c, int stage) {
    uint8_t* const to = mine + stage * R::kStage;
    const int k = c * kFp8Block, cs = min(c, nch - 1);
#pragma unroll
    for (int j = 0; j < DI; ++j) {
      if constexpr (ANY) {
        held[j] = codes16(src[j] + k, lim[j] - k);
      } else {
        const uint8_t* const from = k < lim[j] ? src[j] + k : zeros;
        if (NT && j * 8 >= BM) load_lds16_nt(from, to + (wv * DI + j) * 1024);
        else load_lds16(from, to + (wv * DI + j) * 1024);
      }
    }
#pragma unroll
    for (int j = 0; j < SI; ++j) {
      const float* const from = ssrc[j] ? ssrc[j] + cs : reinterpret_cast<const float*>(zeros);
      if constexpr (ANY) factors[j] = *from;
      else load_lds4(from, to + R::kCodes + (wv + NW * j) * 256);
    }
  };
  auto put = [&](int stage) {
    uint8_t* const to = mine + stage * R::kStage;
#pragma unroll
    for (int j = 0; j < DI; ++j) *reinterpret_cast<uint4*>(to + (wv * DI + j) * 1024 + lane * 16) = held[j];
#pragma unroll
    for (int j = 0; j < SI; ++j)
      *reinterpret_cast<float*>(to + R::kCodes + (wv + NW * j) * 256 + lane * 4) = factors[j];
  };
  floatx4_t acc[TT][FT];
#pragma unroll
  for (int t = 0; t < TT; ++t)
#pragma unroll
    for (int f = 0; f < FT; ++f) acc[t][f] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  const int piece = (kg ^ (li & 7)) * 16;
  const int xat = (wm * TT * 16 + li) * 128, wat = (BM + wn * FT * 16 + (li >> 2) * 4 * FT + (li & 3)) * 128;
  const int sxat = R::kCodes + (wm * TT * 16 + li) * 4, swat = R::kCodes + (BM + wn * FT * 16 / kFp8Block) * 4;
  const int steps = (nch + KW - 1) / KW;
#pragma unroll
  for (int s = 0; s + 1 < ST; ++s) issue(s * KW + kw, s);
  if constexpr (ANY) put(0);
  int st = 0;
  for (int i = 0; i < steps; ++i) {
    // this wave's loads of stage st have landed (its writes are done) and its reads of the stage before, then every
    // wave's
    __builtin_amdgcn_s_waitcnt(vmcnt_only(ANY ? 63 : (ST - 2) * (DI + SI)) & ~0xf00);
    asm volatile("" ::: "memory");
    if constexpr (NW > 1) {
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    }
    const int c = i * KW + kw;
    if constexpr (!kLate) issue(c + (ST - 1) * KW, st == 0 ? ST - 1 : st - 1);
    if (KW == 1 || c < nch) {
      const uint8_t* const from = mine + st * R::kStage;
      auto frag = [&](int at) {
        const int4v u = *reinterpret_cast<const int4v*>(from + at + piece);
        const int4v v = *reinterpret_cast<const int4v*>(from + at + (piece ^ 64));
        return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
      };
      int8v wc[FT], xc[TT];
      float f0[TT];
#pragma unroll
      for (int f = 0; f < FT; ++f) wc[f] = frag(wat + f * 4 * 128);
#pragma unroll
      for (int t = 0; t < TT; ++t) xc[t] = frag(xat + t * 16 * 128);
      const float s = *reinterpret_cast<const float*>(from + swat);
#pragma unroll
      for (int t = 0; t < TT; ++t) f0[t] = *reinterpret_cast<const float*>(from + sxat + t * 64);
      if constexpr (kLate) {
        __builtin_amdgcn_sched_barrier(0);
        issue(c + (ST - 1) * KW, st == 0 ? ST - 1 : st - 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      Operand wf[FT];
#pragma unroll
      for (int f = 0; f < FT; ++f) operand(wc[f], wf[f]);
      floatx4_t p[3];
#pragma unroll
      for (int j = 0; j < TT * FT + 2; ++j) {
        if (j < TT * FT) {
          Operand xf;
          operand(xc[j / FT], xf);
          p[j % 3] = block_sum(wf[j % FT], xf);
        }
        if (j >= 2) {
          const int u = j - 2, t = u / FT, f = u % FT;
          if (f == 0) f0[t] *= s;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][f][e] = __builtin_fmaf(f0[t], p[u % 3][e], acc[t][f][e]);
        }
        if constexpr (kLate && !EXACT) __builtin_amdgcn_sched_barrier(0);
      }
    } else if constexpr (kLate) {
      issue(c + (ST - 1) * KW, st == 0 ? ST - 1 : st - 1);
    }
    st = st + 1 == ST ? 0 : st + 1;
    if constexpr (ANY) put(st);
  }
  // what was requested past the last block must land before the ring is used again or released
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0) & ~0xf00);
  const int col = n0 + wn * FT * 16 + kg * 4 * FT;
  if constexpr (KW == 1) {
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int m = wm * TT * 16 + t * 16 + li;
      if (m < count) {
#pragma unroll
        for (int f = 0; f < FT; ++f) store4(a, m0 + m, col + f * 4, acc[t][f]);
      }
    }
  } else {
    // every group leaves its sums; group i adds up and stores the wave's pieces i, i + KW, ...
    floatx4_t* const sums = reinterpret_cast<floatx4_t*>(ring) + wv * TT * FT * 64 + lane;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TT; ++t)
#pragma unroll
      for (int f = 0; f < FT; ++f) sums[(kw * NW * TT * FT + t * FT + f) * 64] = acc[t][f];
    __syncthreads();
#pragma unroll
    for (int b = 0; b < TT * FT; b += KW) {
      const int i = b + kw;
      if (TT * FT % KW != 0 && i >= TT * FT) break;
      floatx4_t v = sums[i * 64];
#pragma unroll
      for (int k = 1; k < KW; ++k) {
        const floatx4_t u = sums[(k * NW * TT * FT + i) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += u[e];
      }
      const int m = wm * TT * 16 + i / FT * 16 + li;
      if (m < count) store4(a, m0 + m, col + i % FT * 4, v);
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows: 256 tokens x 256 features by 8 waves of 128 x 64, K in blocks through two LDS stages of 64 KB; up to 256
// workgroups go through the tiles.  The one barrier of a block stands before its last two token tiles: all waves'
// fragments of the block are in registers then, so its stage takes the loads of the block after the next, and the
// next block's first fragments are read under the matrix instructions that are left.  Sums are added three
// instructions behind.  The next tile's first two blocks follow this one's last two without a gap.
//
// Bound by the issue of instructions and by power: a wave issues some 216 vector instructions a block, 32 of them
// matrix, and the matrix cores are busy for 47% of the cycles, at 1.9 to 2.0 GHz (LDS 24%).  MI355X: 8,192 x 21,888 x
// 2,048 354 to 363 us (2.02 to 2.07 PFLOP/s), 8,192^3 479 (2.29); 128 x 256 tiles of ring_kernel 552 and 648, but 23 for 31
// with 1,024 x 2,816 x 2,048.  Groups: 49,152 rows of 64, 2,816 x 2,048, 352 to 366 us, 1.17 times their rows in tiles.
// ---------------------------------------------------------------------------
struct Big {
  static constexpr int BM = 256, BN = 256, kThreads = 512, kWgs = 256;
  static constexpr int kStage = (BM + BN) * 128;
  // scales of eight blocks: of the tokens [256][8], the places of tokens 8 i + 8 .. 8 i + 15, i even, exchanged by xor 4
  // (banks), then of the features' two blocks [2][8], four copies; two such windows, and the addresses of the tokens'
  // scales, twice
  static constexpr int kWindow = BM * 32 + 4 * 256, kScales = 2 * kStage, kRows = kScales + 2 * kWindow;
  static constexpr int kGroups = kRows + 2 * BM * 8, kUnused = kGroups + 64 * 12, kLds = kUnused + 8 * 256;
  static_assert(kLds <= 160 * 1024, "LDS");
};

template <bool GROUPED>
__global__ __launch_bounds__(512) void big_kernel(const Args a) {
  constexpr int BM = Big::BM, BN = Big::BN;
  extern __shared__ __attribute__((aligned(16))) uint8_t ring[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1, li = lane & 15, kg = lane >> 4, nch = (a.K + kFp8Block - 1) / kFp8Block;
  const bool gather = GROUPED && a.index, whole = a.wide && a.N % 8 == 0;
  // the tiles of this XCD's workgroups: neighbours in tile_at's order
  int mt = a.mt;
  Groups* const all = reinterpret_cast<Groups*>(ring + Big::kGroups);  // up to 64 groups
  if constexpr (GROUPED) {
    Groups g;
    mt = all_tiles<BM>(a, g);
    if (wave == 0) all[lane] = g;
    __syncthreads();
  }
  const uint32_t total = (uint32_t)mt * a.nt, per = (total + 7) / 8, last = min(((blockIdx.x & 7) + 1) * per, total);
  uint32_t at = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (at >= last) return;

  // the tile whose blocks are requested
  int group = 0, count = 0, n0 = 0;
  int64_t m0 = 0;
  // Loads: waves 0 to 3 the tokens' rows, 4 to 7 the features', 64 each, by offsets that lie past the buffer for what
  // is not there (zeros).  The lane's 16-byte piece of its rows: of even and odd eights of rows, for tokens the same.
  const int at0 = ((lane & 7) ^ (wave < 4 ? lane >> 3 : lane >> 3 & 3)) * 16, at1 = wave < 4 ? at0 : at0 ^ 64;
  constexpr uint32_t kPast = 0x80000000u;
  __amdgpu_buffer_rsrc_t codes;
  uint32_t voff[8];
  uint64_t swrow = 0;  // of waves 4 to 7
  const uint64_t own = wave < 4 ? ~0ull : 0ull;
  // the addresses of the tokens' scales, of this tile and of the next by turns (a slow wave may still read this one's
  // when the next one's are written); for a row that is not there that of a zero, plus 1
  int turn = 0;
  auto srow = [&](int t) { return reinterpret_cast<uint64_t*>(ring + Big::kRows + turn) + t; };
  auto enter = [&](uint32_t tile) {
    int tm, tn;
    // in here: kept over the loop what follows from it is spilled
    int thread = threadIdx.x;
    asm volatile("" : "+v"(thread));
    const int lane = thread & 63;
    tile_at(tile, mt, a.nt, tm, tn);
    if constexpr (GROUPED) {
      group_of<BM>(a, all[lane], tm, group, m0, count);
    } else {
      m0 = (int64_t)tm * BM;
      count = static_cast<int>(min((int64_t)BM, a.rows - m0));
    }
    n0 = tn * BN;
    codes = buffer(wave >= 4 ? a.w + group * a.wgs + n0 * a.ws : gather ? a.x : a.x + m0 * a.xs, kPast);
    const uint32_t stride = static_cast<uint32_t>(wave >= 4 ? a.ws : a.xs);
    const int rows = wave >= 4 ? a.N - n0 : count;
    if (gather && wave < 4) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = wave * 64 + j * 8 + (lane >> 3), r = i < rows ? a.index[m0 + i] : -1;
        voff[j] = r >= 0 && r < a.xrows ? r * stride + (j & 1 ? at1 : at0) : kPast;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = (wave & 3) * 64 + j * 8 + (lane >> 3);
        voff[j] = i < rows ? i * stride + (j & 1 ? at1 : at0) : kPast;
      }
    }
    swrow = ~own & reinterpret_cast<uint64_t>(
                       a.sw + group * a.swgs + min(n0 / kFp8Block + (lane >> 3 & 1), (a.N - 1) / kFp8Block) * a.sws);
    turn ^= BM * 8;
    if (thread < BM) {
      int64_t row = thread < count ? m0 + thread : -1;
      if (gather && row >= 0) row = a.index[row];
      *srow(thread) = row < 0 || row >= a.xrows ? reinterpret_cast<uint64_t>(kZeros) + 1
                                                : reinterpret_cast<uint64_t>(a.sx + row * a.sxs);
    }
  };
  // pieces past the rows' end: of the last block, which is the tile's last to be requested
  auto cut = [&] {
    const int k = (nch - 1) * kFp8Block;
#pragma unroll
    for (int j = 0; j < 8; ++j) voff[j] |= k + (j & 1 ? at1 : at0) < a.K ? 0u : kPast;
  };
  // no branch in these two: in the middle of a block's instructions one costs the loop over 100 spilled registers
  auto issue = [&](int c, int stage) {
    uint8_t* const to = ring + stage * Big::kStage;
#pragma unroll
    for (int j = 0; j < 8; ++j) buffer_lds16(codes, to + (wave * 8 + j) * 1024, voff[j], c * kFp8Block);
  };
  // an eighth of a window: waves 0 to 3 eight tokens' scales each, the others the features' (each its own copy)
  const int swap = wave < 4 ? (wave & 1) << 2 : 0;
  auto scales = [&](int part, int window0) {  // part: counted over the tile's windows
    const int in = part & 7, first = part & ~7, t = in * 32 + (wave & 3) * 8 + (lane >> 3);
    const uint64_t row = *srow(t) & own | swrow;
    const int b = row & 1 ? 0 : min(first + ((lane & 7) ^ swap), nch - 1);
    const int window = Big::kScales + ((part >> 3) + window0 & 1) * Big::kWindow;
    const int to = wave < 4 ? (in * 4 + wave) * 256 : BM * 32 + (wave - 4) * 256;
    // a window past the last block's goes where nothing is read, not into the next tile's first
    load_lds4(reinterpret_cast<const float*>(row & ~1ull) + b,
              ring + (first < nch ? window + to : Big::kUnused + wave * 256));
  };
  floatx4_t acc[8][4];
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int f = 0; f < 4; ++f) acc[t][f] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  const int piece = (kg ^ (li & 7)) * 16;
  const int xat = (wm * 128 + li) * 128, wat = (BM + wn * 64 + (li >> 2) * 8 + (li & 3)) * 128;
  const int sxat = (wm * 128 + li) * 32, sxkey = li >> 3 << 2, swat = BM * 32 + (wn >> 1) * 32;
  auto frag = [&](const uint8_t* from, int at) {
    const int4v u = *reinterpret_cast<const int4v*>(from + at + piece);
    const int4v v = *reinterpret_cast<const int4v*>(from + at + (piece ^ 64));
    return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  // This wave's loads have landed and its reads are done, then every wave's.  Behind a tile's end its 16 stores may be on
  // their way still (the branch is written out: the compiler's would cut the block's instructions in two).
  int stores = 0;
  auto meet = [&] {
    asm volatile(
        "s_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 .Lstores%=\n\ts_waitcnt vmcnt(0)\n.Lstores%=:\n\t"
        "s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::"s"(stores)
        : "memory", "scc");
  };
  int8v wf[4], xf[3];
  float nx[8], nw;
  auto read_scales = [&](int c, int window0) {
    const uint8_t* const win = ring + Big::kScales + ((c >> 3) + window0 & 1) * Big::kWindow;
#pragma unroll
    for (int t = 0; t < 8; ++t) nx[t] = *reinterpret_cast<const float*>(win + sxat + ((c & 7) ^ sxkey) * 4 + t * 512);
    nw = *reinterpret_cast<const float*>(win + swat + (c & 7) * 4);
  };
  auto read_w = [&](const uint8_t* from, int f) { wf[f] = frag(from, wat + (f >> 1) * 4096 + (f & 1) * 512); };
  enter(at);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 9; ++i) scales(i, 0);
  issue(0, 0);
  meet();
  if (nch == 2) cut();
  issue(1, 1);
  int stage = 0, window = 0;  // the block's stage, the tile's first window's place
  int kc = 2, kwin = 0;       // the block that is requested (of this tile or the next), its tile's first window
  read_scales(0, 0);
#pragma unroll
  for (int f = 0; f < 4; ++f) read_w(ring, f);
  xf[0] = frag(ring, xat);
  xf[1] = frag(ring, xat + 2048);
  // the sums on their way: of the last three instructions, added in the next block
  floatx4_t p[4];
  float sx7 = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  for (;;) {
    const int64_t om0 = m0;
    const int ocount = count, on0 = n0;
    for (int c = 0; c < nch; ++c) {
      if (c == nch - 2) {  // what is requested from here on is the next tile's
        at += (gridDim.x + 7) >> 3;
        kc = 0;
        kwin = window + ((nch - 1) >> 3) + 1 & 1;  // not where this tile's last scales are
        if (at < last) {
          enter(at);
          __builtin_amdgcn_s_waitcnt(vmcnt_only(63) & ~0xf00);
          __builtin_amdgcn_s_barrier();  // the scales' addresses are written
          asm volatile("" ::: "memory");
#pragma unroll
          for (int i = 0; i < 7; ++i) scales(i, kwin);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) voff[j] = kPast;
        }
      }
      if (kc == nch - 1) cut();
      const uint8_t* const from = ring + stage * Big::kStage;
      const uint8_t* const next = ring + (stage ^ 1) * Big::kStage;
      const bool end = c + 1 == nch;
      float sx[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) sx[t] = nx[t] * nw;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int t = i >> 2, f = i & 3;
        __builtin_amdgcn_sched_barrier(0);
        p[i & 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[f], xf[t % 3], floatx4_t{0.f, 0.f, 0.f, 0.f}, 0, 0,
                                                                    0, 0, 0, 0);
        if (f == 0 && t < 6) xf[(t + 2) % 3] = frag(from, xat + (t + 2) * 2048);
        if (i == 23) {
          meet();
          stores = 0;
          issue(kc, stage);
        }
        if (i == 24) scales(kc + 7, kwin);
        // the next block's first fragments, each behind the last use of the one whose place it takes
        if (i == 25) read_scales(end ? 0 : c + 1, end ? kwin : window);
        if (i == 28) xf[0] = frag(next, xat);
        if (i >= 29) read_w(next, i - 29);
        if (i == 31) {
          read_w(next, 3);
          xf[1] = frag(next, xat + 2048);
        }
        const int tt = i >= 3 ? (i - 3) >> 2 : 7, ff = (i - 3) & 3;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[tt][ff][e] = __builtin_fmaf(i >= 3 ? sx[tt] : sx7, p[(i - 3) & 3][e], acc[tt][ff][e]);
      }
      __builtin_amdgcn_sched_barrier(0);
      sx7 = sx[7];
      stage ^= 1;
      ++kc;
    }
    window = kwin;
#pragma unroll
    for (int f = 1; f < 4; ++f)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[7][f][e] = __builtin_fmaf(sx7, p[f][e], acc[7][f][e]);
    // the next tile's first block adds these once more: nothing of them may be left, a NaN would outlast a factor of zero
    sx7 = 0.f;
#pragma unroll
    for (int f = 1; f < 4; ++f) p[f] = floatx4_t{0.f, 0.f, 0.f, 0.f};
    // lane group kg holds features 8 kg .. 8 kg + 7 of each half of the wave's 64
    int r0 = wm * 128 + li;
    asm volatile("" : "+v"(r0));  // here: kept over the loop the rows' offsets are spilled, and a reload waits for the stores
    const int col = on0 + wn * 64 + kg * 8;
    auto pair = [&](int t, int i) {
      const floatx4_t u = acc[t][2 * i], v = acc[t][2 * i + 1];
      return u32x4_t{pack2(u[0], u[1]), pack2(u[2], u[3]), pack2(v[0], v[1]), pack2(v[2], v[3])};
    };
    if (whole) {
      // as many stores for every wave, so that the next block's wait may leave them on their way; what is not the
      // tile's lies past the buffer
      const __amdgpu_buffer_rsrc_t out = buffer(static_cast<bf16_t*>(a.y) + om0 * a.ys, kPast);
      const uint32_t out0 = col < a.N ? col * 2 : kPast, out1 = col + 32 < a.N ? col * 2 + 64 : kPast;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int m = r0 + t * 16;
        const uint32_t row = m < ocount ? m * (uint32_t)a.ys * 2 : kPast;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          __builtin_amdgcn_raw_buffer_store_b128(pair(t, i), out,
                                                 row + (i ? out1 : out0) | (row | (i ? out1 : out0)) & kPast, 0, 0);
      }
      stores = 16;
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int m = r0 + t * 16;
        if (m < ocount) {
          bf16_t* const row = static_cast<bf16_t*>(a.y) + (om0 + m) * a.ys;
#pragma unroll
          for (int i = 0; i < 2; ++i) store8_any(row, col + 32 * i, a.N, pair(t, i));
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int f = 0; f < 4; ++f) acc[t][f] = floatx4_t{0.f, 0.f, 0.f, 0.f};
    if (at >= last) break;
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // what was requested past the last block must land before the ring is released
}

// ---------------------------------------------------------------------------
// Which of them.  A launch of up to 256 tiles (one a CU) takes about a + b k us, k the blocks of K, and each further
// round of them c + d k more; the last round takes as long with one tile as with 256.  (Measured on MI355X: 135 products
// of 1 to 4,096 rows, 512 to 10,944 columns, off by 3 to 8% on the mean.  The shape that is taken was 0.4% slower
// on the mean than the best one, with fp32 results 1%; estimates without whole rounds 7%.)  Groups' tiles also wait for
// memory: what they load together takes at least 3 us and 8 TB/s (31 products of 4 to 4,000 tokens of 8 to 128
// groups: 2% slower than the best, without this 5%).
// ---------------------------------------------------------------------------
constexpr int64_t kStreamed = 64ll << 20;
struct Cost {
  int bm, bn, threads;  // of a workgroup
  float a, b, c, d;
};
enum Shape { kFew, kFew32, kTall32, kWide32, kMid, kMid128, kTile128, kLong128, kBig, kShapes, kStream, kAny };
constexpr Cost kCost[kShapes] = {
    {16, 16, 512, 2.85f, 0.069f, 0.81f, 0.043f},     // 8 waves along K
    {32, 16, 512, 3.22f, 0.083f, 1.78f, 0.071f},     // 8 along K
    {32, 32, 256, 2.71f, 0.149f, 0.83f, 0.093f},     // 4 along K
    {32, 64, 128, 3.11f, 0.333f, 0.83f, 0.135f},     // 2 along K
    {64, 64, 512, 3.92f, 0.275f, 2.31f, 0.269f},     // 4 on the tile, 2 along K
    {128, 64, 512, 4.45f, 0.446f, 3.18f, 0.438f},    // 4 on the tile, 2 along K
    {128, 128, 512, 4.75f, 0.671f, 3.35f, 0.704f},   // 8 on the tile
    {128, 256, 1024, 6.42f, 0.965f, 7.45f, 1.024f},  // 16 on the tile (fp32 results: 8)
    {256, 256, 512, 7.28f, 1.525f, 6.08f, 1.588f},   // big_kernel
};
constexpr Cost kStreamed32 = {16, 32, 64, 0.f, 0.f, 0.f, 0.f};  // chosen by another rule
constexpr const Cost& tile_of_shape(int s) { return s == kStream ? kStreamed32 : kCost[s % kAny]; }
constexpr int threads_of(int s, bool f32) { return s == kLong128 && f32 ? 512 : tile_of_shape(s).threads; }

// token tiles: the most there may be, and as many as are likely (groups of like sizes)
int64_t most_tiles(const Args& a, bool grouped, int bm) {
  return grouped ? (a.rows + min(a.rows, (int64_t)a.groups) * (bm - 1)) / bm : (a.rows + bm - 1) / bm;
}
float likely_tiles(const Args& a, bool grouped, int bm) {
  if (!grouped) return static_cast<float>((a.rows + bm - 1) / bm);
  const float rows = static_cast<float>(a.rows), hit = a.groups * (1.f - expf(-rows / a.groups));
  return fmaxf(hit, rows / bm + 0.5f * hit);
}

// a launch has fewer than 2^32 threads
bool launchable(const Args& a, bool grouped, int shape) {
  const Cost& c = tile_of_shape(shape);
  return most_tiles(a, grouped, c.bm) <=
         ((1ll << 32) / threads_of(shape, a.out_f32) - 8) / ((a.N + (int64_t)c.bn - 1) / c.bn);
}

// the least estimate among the shapes whose bits are set and that have not too many tiles
Shape choose(const Args& a, bool grouped, unsigned among) {
  const float k = static_cast<float>((a.K + kFp8Block - 1) / kFp8Block);
  Shape best = kFew;
  float least = 3e38f;
  for (int s = 0; s < kShapes; ++s) {
    if (!(among >> s & 1)) continue;
    const Cost& c = kCost[s];
    if (!launchable(a, grouped, s)) continue;
    const float n = likely_tiles(a, grouped, c.bm) * ((a.N + c.bn - 1) / c.bn);
    float t = c.a + c.b * k + fmaxf(ceilf(n * (1.f / 256)) - 1.f, 0.f) * (c.c + c.d * k);
    if (grouped) t = fmaxf(t, 3.f + n * (c.bm + c.bn) * a.K * (1.f / 8e6f));
    if (t < least) least = t, best = static_cast<Shape>(s);
  }
  return best;
}

bool set_tiles(Args& a, bool grouped, int shape) {
  const Cost& c = tile_of_shape(shape);
  a.mt = (int)most_tiles(a, grouped, c.bm);
  a.nt = (a.N + c.bn - 1) / c.bn;
  if (launchable(a, grouped, shape)) return true;
  dsv2_set_error("linear_fp8_blocks: %lld rows of %d", (long long)a.rows, a.N);
  return false;
}
dim3 grid_of(const Args& a) { return dim3((unsigned)(((int64_t)a.mt * a.nt + 7) / 8 * 8)); }

template <int SHAPE, int WM, int WN, int TT, int FT, int KW, int ST, bool NT, bool ANY, bool EXACT, bool GROUPED>
int launch_ring(Args a, hipStream_t st) {
  using R = Ring<WM, WN, TT, FT, KW, ST>;
  static_assert(R::BM == tile_of_shape(SHAPE).bm && R::BN == tile_of_shape(SHAPE).bn &&
                R::kThreads == threads_of(SHAPE, EXACT), "what the choice goes by");
  if (!set_tiles(a, GROUPED, SHAPE)) return DSV2_E_SHAPE;
  ring_kernel<WM, WN, TT, FT, KW, ST, NT, ANY, EXACT, GROUPED><<<grid_of(a), R::kThreads, R::kLds, st>>>(a);
  return dsv2_launch_status(GROUPED ? "grouped_linear_fp8_blocks" : "linear_fp8_blocks");
}

template <bool GROUPED>
int launch_big(Args a, hipStream_t st) {
  static_assert(Big::BM == kCost[kBig].bm && Big::BN == kCost[kBig].bn && Big::kThreads == kCost[kBig].threads, "the same");
  if (!set_tiles(a, GROUPED, kBig)) return DSV2_E_SHAPE;
  dim3 grid = grid_of(a);
  grid.x = min(grid.x, (unsigned)Big::kWgs);
  big_kernel<GROUPED><<<grid, Big::kThreads, Big::kLds, st>>>(a);
  return dsv2_launch_status(GROUPED ? "grouped_linear_fp8_blocks" : "linear_fp8_blocks");
}

// the tiles of a call; kAny is added where its rows go through registers
int shape_of(const Args& a, bool grouped) {
  if (a.K % 16 != 0 || !dsv2_aligned16(a.x) || !dsv2_aligned16(a.w) || a.xs % 16 != 0 || a.ws % 16 != 0 || a.wgs % 16 != 0)
    return kAny + choose(a, grouped, 1 << kFew | 1 << kTall32 | 1 << kMid | 1 << kTile128);
  // Weights that are read once and do not stay in the 256 MB of the last-level cache (a model's others are read in
  // between): one wave a tile, many workgroups a CU, and the non-temporal hint (MI355X: 5 x 102,400 x 2,048, fp32, 36.6
  // us, 5.8 TB/s, the best of the others 49.6; 64 tokens x 6 of 64 groups of 2,816 x 2,048 62.4 / 75.6).  Smaller ones
  // the other way: 64 x 2,048 x 10,944 (22 MB) 30 / 11, 1 x 3,648 x 2,048 (7 MB) 8 / 3.5.  Groups go by their mean, which
  // is all that the host knows: 1,020 rows of 64 groups 94 us where most groups have some, 48 where one has them all.
  if (a.rows <= 16 * (grouped ? (int64_t)a.groups : 1) && (int64_t)a.groups * a.N >= (kStreamed + a.K - 1) / a.K &&
      launchable(a, grouped, kStream))
    return kStream;
  // big_kernel's offsets are 31 bits: those of its tile's rows, or of all of x where rows are taken by number
  constexpr int64_t kReach = 1ll << 31;
  const bool big = !a.out_f32 && a.K > kFp8Block && 256 * a.ws + a.K < kReach &&
                   512 * a.ys < kReach && (a.index ? a.xrows : 256) * a.xs + a.K < kReach;
  return choose(a, grouped, (1 << kShapes) - 1 - (big ? 0 : 1 << kBig));
}

template <bool EXACT, bool GROUPED>
int launch(const Args& a, hipStream_t st) {
  switch (shape_of(a, GROUPED)) {
    case kFew: return launch_ring<kFew, 1, 1, 1, 1, 8, 2, false, false, EXACT, GROUPED>(a, st);
    case kFew32: return launch_ring<kFew32, 1, 1, 2, 1, 8, 2, false, false, EXACT, GROUPED>(a, st);
    case kTall32: return launch_ring<kTall32, 1, 1, 2, 2, 4, 2, false, false, EXACT, GROUPED>(a, st);
    case kWide32: return launch_ring<kWide32, 1, 1, 2, 4, 2, 2, false, false, EXACT, GROUPED>(a, st);
    case kMid: return launch_ring<kMid, 2, 2, 2, 2, 2, 3, false, false, EXACT, GROUPED>(a, st);
    case kMid128: return launch_ring<kMid128, 2, 2, 4, 2, 2, 3, false, false, EXACT, GROUPED>(a, st);
    case kTile128: return launch_ring<kTile128, 2, 4, 4, 2, 1, 4, false, false, EXACT, GROUPED>(a, st);
    case kLong128: return launch_ring<kLong128, EXACT ? 2 : 4, 4, EXACT ? 4 : 2, 4, 1, 3, false, false, EXACT, GROUPED>(a, st);
    case kStream: return launch_ring<kStream, 1, 1, 1, 2, 1, 3, true, false, EXACT, GROUPED>(a, st);
    case kAny + kFew: return launch_ring<kAny + kFew, 1, 1, 1, 1, 8, 2, false, true, EXACT, GROUPED>(a, st);
    case kAny + kTall32: return launch_ring<kAny + kTall32, 1, 1, 2, 2, 4, 2, false, true, EXACT, GROUPED>(a, st);
    case kAny + kMid: return launch_ring<kAny + kMid, 2, 2, 2, 2, 2, 2, false, true, EXACT, GROUPED>(a, st);
    case kAny + kTile128: return launch_ring<kAny + kTile128, 2, 4, 4, 2, 1, 2, false, true, EXACT, GROUPED>(a, st);
    default: break;
  }
  if constexpr (!EXACT) return launch_big<GROUPED>(a, st);
  else return DSV2_E_FLAGS;  // not reached: kBig is for bf16 results
}

bool aligned(const void* p, int to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace

#define CHECK_PRODUCT(name)                                                                                       \
  DSV2_REQUIRE(out_dtype == DSV2_DTYPE_BF16 || out_dtype == DSV2_DTYPE_F32, DSV2_E_FLAGS, name ": out_dtype %d", \
               out_dtype);                                                                                        \
  DSV2_REQUIRE(rows >= 0 && rows <= 0x7fffffff && K > 0 && K <= 1 << 30 && N > 0 && N <= 1 << 30, DSV2_E_SHAPE, \
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
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return a.out_f32 ? launch<true, false>(a, st) : launch<false, false>(a, st);
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
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return a.out_f32 ? launch<true, true>(a, st) : launch<false, true>(a, st);
}

int dsv2_linear_fp8_blocks_tiles(int64_t rows, int K, int N, int groups, int out_dtype) {
  DSV2_REQUIRE(rows > 0 && rows <= 0x7fffffff && K > 0 && K <= 1 << 30 && N > 0 && N <= 1 << 30 && groups >= 0 &&
                   groups <= 65536, DSV2_E_SHAPE, "linear_fp8_blocks_tiles: %lld rows, K %d, N %d, %d groups",
               (long long)rows, K, N, groups);
  Args a{};
  a.xs = a.ws = K;
  a.wgs = (int64_t)N * K;
  a.ys = N;
  a.rows = a.xrows = rows;
  a.K = K;
  a.N = N;
  a.groups = groups > 0 ? groups : 1;
  a.out_f32 = out_dtype == DSV2_DTYPE_F32;
  a.wide = (int64_t)N * (a.out_f32 ? 4 : 2) % 16 == 0;
  return shape_of(a, groups > 0);
}
