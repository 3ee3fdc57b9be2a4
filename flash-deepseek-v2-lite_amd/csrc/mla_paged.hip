// Absorbed-MLA attention over the paged latent cache held in 4 bits.
//
//   s_t = scale * q . (latent_t | rope_t),  p = softmax(s),  o = sum_t p_t latent_t
//
// One (query token, head) pair is a column; a request's columns are numbered token by token, and 16 of
// them make the narrow side of v_mfma_f32_16x16x32_bf16 (S^T = K Q^T, O^T += V^T P^T).  An item is one
// request and 16 of its columns: ceil(length / 32) tiles of 32 tokens.
//
// Work is dealt out on the device, where the lengths are: every workgroup sums the items' tiles for
// itself and takes an equal run of them, whatever requests it crosses.  An item that lies within one
// workgroup is finished there; of one that crosses into others each leaves its part (fp32 o, max, sum)
// in the workspace and mla_paged_merge_kernel joins them.
#include "paged.h"

using namespace paged;

namespace {
constexpr int kTile = 32;
constexpr int kWaves = 4;
constexpr int kVRow = kLat + 16;       // padded LDS row of a token's latent (elements): 1,056 bytes
constexpr int kORow = kLat + 4;        // padded LDS row of a column's output (floats)
constexpr int kWaveLds = kTile * kVRow * 2;
static_assert(16 * kORow * 4 <= kWaveLds, "a wave's outputs take its tile's place");
constexpr int kWgs = 256;              // one workgroup per CU
constexpr int kMinTiles = 8;           // tiles of a workgroup, at least
constexpr int kMaxRequests = 4096;     // the running tile counts stand in LDS
constexpr int kPartFloats = 16 * kLat;

struct PagedAttnArgs {
  const bf16_t* q;
  int64_t q_ts, q_hs;
  int tokens, heads;
  const uint8_t* pages;
  int64_t page_stride;
  int n_pages, shift;
  const int32_t* table;
  int64_t ts;
  int width;
  const int32_t* lens;
  const int32_t* cu_q;
  int max_q;
  int requests;
  int columns16;  // most column groups of a request
  float scale_log2;
  bf16_t* out;
  int64_t o_ts, o_hs;
  float* part_o;     // [2 * kWgs][16][512]
  float* part_ml;    // [2 * kWgs][16][2]
  int32_t* starts;   // [requests * columns16 + 1]: an item's first tile; last: tiles of a workgroup
  int32_t* status;
};

struct Request {
  int len, q0, nq, columns;
};
__device__ __forceinline__ Request request(const PagedAttnArgs& a, int b) {
  Request r;
  const int64_t room = static_cast<int64_t>(a.width) << a.shift;
  r.len = static_cast<int>(min(static_cast<int64_t>(max(a.lens[b], 0)), room));
  r.q0 = b;
  r.nq = 1;
  if (a.cu_q) {
    r.q0 = a.cu_q[b];
    r.nq = r.q0 >= 0 ? max(min(a.cu_q[b + 1], a.tokens) - r.q0, 0) : 0;
  }
  r.columns = min(r.nq, a.max_q) * a.heads;
  return r;
}

// a tile's bytes: lane (li, kg) has 16-token blocks h = 0, 1's token li, latent blocks 4c + kg (32 codes
// each), the token's 16 scales, rotary keys y * 32 + kg * 8 .. +8
struct Raw {
  uint4 code[2][4];
  uint4 rope[2][2];
  uint4 scale[2];
  bool ok[2];  // the token exists and its page is one
};
}  // namespace

__global__ __launch_bounds__(64 * kWaves, 1) void mla_paged_kernel(const PagedAttnArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ float ml[kWaves][16][2];
  __shared__ int32_t wave_sum32[kWaves];
  int32_t* ends = reinterpret_cast<int32_t*>(smem + kWaves * kWaveLds);
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, li = lane & 15, kg = lane >> 4;

  // running tile counts of the requests (the host has checked that they stay within int32)
  int total;
  {
    const int per = (a.requests + 255) / 256;
    const int b0 = min(tid * per, a.requests), b1 = min(b0 + per, a.requests);
    int run = 0;
    for (int b = b0; b < b1; ++b) {
      const Request r = request(a, b);
      if (r.nq > a.max_q && blockIdx.x == 0 && a.status) atomicOr(a.status, DSV2_DEVERR_TOKENS);
      run += ((r.len + kTile - 1) / kTile) * ((r.columns + 15) / 16);
      ends[b] = run;
    }
    int scan = run;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(scan, o, DSV2_WAVE);
      if (lane >= o) scan += u;
    }
    if (lane == 63) wave_sum32[wv] = scan;
    __syncthreads();
    int before = scan - run;
    total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i < wv) before += wave_sum32[i];
      total += wave_sum32[i];
    }
    for (int b = b0; b < b1; ++b) ends[b] += before;
    __syncthreads();
  }
  const int per = max((total + kWgs - 1) / kWgs, kMinTiles);
  if (blockIdx.x == 0 && tid == 0) a.starts[a.requests * a.columns16] = per;
  const int64_t from = static_cast<int64_t>(blockIdx.x) * per;
  if (from >= total) return;
  const int first = static_cast<int>(from), last = min(first + per, total);
  int b;
  {
    int lo = 0, hi = a.requests - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > first)
        hi = mid;
      else
        lo = mid + 1;
    }
    b = lo;
  }

  bf16_t* const vt = reinterpret_cast<bf16_t*>(smem + wv * kWaveLds);
  for (int at = first; at < last;) {
    while (ends[b] <= at) ++b;
    const Request r = request(a, b);
    const int tiles = (r.len + kTile - 1) / kTile;
    const int b_start = b ? ends[b - 1] : 0;
    const int ct = (at - b_start) / tiles;
    const int item = b_start + ct * tiles;  // its first tile
    const int t_first = at - item, t_last = min(last - item, tiles);
    const int col = ct * 16 + li;
    const bool live = col < r.columns;
    const int j = live ? col / a.heads : 0, h = live ? col - j * a.heads : 0;
    const int seen = live ? max(r.len - r.nq + j + 1, 0) : 0;

    // Q^T fragments (B operand): column li; the k order of a block group's four products is the lanes'
    // own: k-slot (kg, e) of product (c, x) is latent (4c + kg) * 32 + x * 8 + e
    bf16x8_t qf[18];
    {
      const bf16_t* qc = a.q + (r.q0 + j) * a.q_ts + h * a.q_hs;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        qf[i] = as_bf16x8(keep_if(live, ldg16(qc + ((i >> 2) * 4 + kg) * 32 + (i & 3) * 8)));
#pragma unroll
      for (int y = 0; y < 2; ++y) qf[16 + y] = as_bf16x8(keep_if(live, ldg16(qc + kLat + y * 32 + kg * 8)));
    }

    const int32_t* row = a.table + b * a.ts;
    auto load_pages = [&](int tile, int* pg) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) pg[hf] = row[min(tile * kTile + hf * 16 + li, r.len - 1) >> a.shift];
    };
    auto load_tile = [&](int tile, const int* pg, Raw& w) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int t = tile * kTile + hf * 16 + li;
        const bool page = pg[hf] >= 0 && pg[hf] < a.n_pages;
        w.ok[hf] = page && t < r.len;
        if (!page && kg == 0 && t < r.len && a.status) atomicOr(a.status, DSV2_DEVERR_BAD_SLOT);
        const int off = min(t, r.len - 1) & ((1 << a.shift) - 1);
        const uint8_t* base = a.pages + (page ? pg[hf] : 0) * a.page_stride;
        const uint8_t* code = base + off * kCodeB + kg * 16;
#pragma unroll
        for (int c = 0; c < 4; ++c) w.code[hf][c] = ldg16(code + c * 64);
        const uint8_t* rope = base + (kCodeB << a.shift) + off * kRopeB + kg * 16;
#pragma unroll
        for (int y = 0; y < 2; ++y) w.rope[hf][y] = ldg16(rope + y * 64);
        w.scale[hf] = ldg16(base + ((kCodeB + kRopeB) << a.shift) + off * kScaleB);
      }
    };

    float m_run = -__FLT_MAX__, l_run = 0.f;
    floatx4_t acc[32];
#pragma unroll
    for (int f = 0; f < 32; ++f) acc[f] = floatx4_t{0.f, 0.f, 0.f, 0.f};

    auto tile_step = [&](int tile, Raw& w) {
      floatx4_t sc[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        uint32_t s[4];
        const uint32_t sw[4] = {w.scale[hf].x, w.scale[hf].y, w.scale[hf].z, w.scale[hf].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) s[c] = (sw[c] >> (8 * kg)) & 0xff;
        // rare: a token past the end or on no page (zeros), a block of NaN (its codes are zeros; one
        // rotary key becomes NaN instead, so that only the queries that see the token get NaN: a NaN
        // latent times an unseen token's p = 0 would be one too)
        const bool nan = max(max(s[0], s[1]), max(s[2], s[3])) == kNanScale;
        if (__any(!w.ok[hf] || nan)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            w.code[hf][c] = keep_if(w.ok[hf] && s[c] != kNanScale, w.code[hf][c]);
            s[c] = w.ok[hf] && s[c] != kNanScale ? s[c] : 127;
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) w.rope[hf][y] = keep_if(w.ok[hf], w.rope[hf][y]);
          if (nan && w.ok[hf]) w.rope[hf][0].x = 0x7fc07fc0u;
        }
        sc[hf] = floatx4_t{0.f, 0.f, 0.f, 0.f};
        bf16_t* vr = vt + (hf * 16 + li) * kVRow + kg * 32;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t cw[4] = {w.code[hf][c].x, w.code[hf][c].y, w.code[hf][c].z, w.code[hf][c].w};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint4 v = decode8(cw[x], s[c]);
            *reinterpret_cast<uint4*>(vr + c * 128 + x * 8) = v;
            sc[hf] = mfma16x16x32(as_bf16x8(v), qf[c * 4 + x], sc[hf]);
          }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) sc[hf] = mfma16x16x32(as_bf16x8(w.rope[hf][y]), qf[16 + y], sc[hf]);
      }
      asm volatile("" ::: "memory");
      float p[8], mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = tile * kTile + (i >> 2) * 16 + 4 * kg + (i & 3) < seen ? sc[i >> 2][i & 3] : -INFINITY;
        mx = fmaxf(mx, p[i]);
      }
      mx = xor32_max(xor16_max(mx)) * a.scale_log2;
      // lazy rescaling: the running maximum (log2 units) moves, and o and l are rescaled, only where a
      // tile exceeds it by more than 8, so p <= 256; it starts below every finite score
      const bool grow = mx > m_run + 8.f;
      if (__any(grow)) {
        const float m_new = grow ? mx : m_run;
        const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
        m_run = m_new;
#pragma unroll
        for (int f = 0; f < 32; ++f) acc[f] *= alpha;
      }
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i], a.scale_log2, -m_run));
        sum += p[i];
      }
      l_run += sum;  // this lane's tokens; the lanes meet at the end
      // P^T (B operand): column li, tokens 4 kg + e then 16 + 4 kg + e; the V^T fragments take the same
      // tokens through two transposed reads (lane (li, kg) addresses token 4 kg + li / 4)
      const bf16x8_t pb = as_bf16x8(pack8(p));
      const bf16_t* vp = vt + (4 * kg + (li >> 2)) * kVRow + 4 * (li & 3);
#pragma unroll
      for (int f = 0; f < 32; ++f) {
        const uint2 lo = lds_read_tr16(vp + f * 16), hi = lds_read_tr16(vp + f * 16 + 16 * kVRow);
        acc[f] = mfma16x16x32(as_bf16x8(make_uint4(lo.x, lo.y, hi.x, hi.y)), pb, acc[f]);
      }
      asm volatile("" ::: "memory");
    };

    // wave w takes tiles t_first + w, + 4, ...: one ahead in registers, its pages one further
    {
      const int end = t_last - 1;
      int tile = t_first + wv;
      int pg[2];
      Raw w0, w1;
      load_pages(min(tile, end), pg);
      load_tile(min(tile, end), pg, w0);
      load_pages(min(tile + kWaves, end), pg);
      while (tile < t_last) {
        load_tile(min(tile + kWaves, end), pg, w1);
        load_pages(min(tile + 2 * kWaves, end), pg);
        tile_step(tile, w0);
        tile += kWaves;
        if (tile >= t_last) break;
        load_tile(min(tile + kWaves, end), pg, w0);
        load_pages(min(tile + 2 * kWaves, end), pg);
        tile_step(tile, w1);
        tile += kWaves;
      }
    }
    l_run = xor32_sum(xor16_sum(l_run));

    // the waves' parts meet in LDS, in each wave's own tile's place
    if (kg == 0) {
      ml[wv][li][0] = m_run;
      ml[wv][li][1] = l_run;
    }
    __syncthreads();
    float m_all = ml[0][li][0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) m_all = fmaxf(m_all, ml[i][li][0]);
    {
      const float weight = __builtin_amdgcn_exp2f(m_run - m_all);
      float* o = reinterpret_cast<float*>(smem + wv * kWaveLds) + li * kORow + 4 * kg;
#pragma unroll
      for (int f = 0; f < 32; ++f) {
        const floatx4_t v = acc[f] * weight;
        *reinterpret_cast<float4*>(o + f * 16) = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    __syncthreads();
    const bool whole = t_first == 0 && t_last == tiles;
    const int slot = at == first ? 2 * blockIdx.x : 2 * blockIdx.x + 1;
    if (t_first == 0 && tid == 0) a.starts[b * a.columns16 + ct] = item;
#pragma unroll
    for (int i = 0; i < kPartFloats / 4 / 256; ++i) {
      const int f = tid + 256 * i, c = f >> 7, d = (f & 127) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < kWaves; ++u) {
        const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + u * kWaveLds) + c * kORow + d);
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
      }
      if (!whole) {
        *reinterpret_cast<float4*>(a.part_o + static_cast<int64_t>(slot) * kPartFloats + c * kLat + d) = v;
        continue;
      }
      const int cc = ct * 16 + c;
      if (cc >= r.columns) continue;
      float mm = ml[0][c][0], l = 0.f;
#pragma unroll
      for (int u = 1; u < kWaves; ++u) mm = fmaxf(mm, ml[u][c][0]);
#pragma unroll
      for (int u = 0; u < kWaves; ++u) l += ml[u][c][1] * __builtin_amdgcn_exp2f(ml[u][c][0] - mm);
      const int jj = cc / a.heads, hh = cc - jj * a.heads;
      const float inv = r.len - r.nq + jj + 1 > 0 ? 1.0f / l : 0.f;
      *reinterpret_cast<uint2*>(a.out + (r.q0 + jj) * a.o_ts + hh * a.o_hs + d) =
          make_uint2(pack2(v.x * inv, v.y * inv), pack2(v.z * inv, v.w * inv));
    }
    if (!whole && tid < 16) {
      float mm = ml[0][tid][0], l = 0.f;
#pragma unroll
      for (int u = 1; u < kWaves; ++u) mm = fmaxf(mm, ml[u][tid][0]);
#pragma unroll
      for (int u = 0; u < kWaves; ++u) l += ml[u][tid][1] * __builtin_amdgcn_exp2f(ml[u][tid][0] - mm);
      a.part_ml[(slot * 16 + tid) * 2] = mm;
      a.part_ml[(slot * 16 + tid) * 2 + 1] = l;
    }
    at = item + t_last;
    if (at < last) __syncthreads();  // the next item's tiles and maxima go where these were read
  }
}

// One workgroup per item, column and quarter of the features: joins the parts of an item that crossed
// workgroups, writes zeros for a request with nothing cached, leaves finished items alone.  8 groups of 32
// threads (4 features each) take every eighth part.
__global__ __launch_bounds__(256) void mla_paged_merge_kernel(const PagedAttnArgs a) {
  __shared__ float wgt[2 * kWgs];
  __shared__ float red[8];
  __shared__ float4 osum[8][32];
  const int b = blockIdx.x / a.columns16, ct = blockIdx.x % a.columns16, c = blockIdx.y, tid = threadIdx.x;
  const int lane = tid & 63, wv = tid >> 6;
  const Request r = request(a, b);
  const int cc = ct * 16 + c;
  if (cc >= r.columns) return;
  const int j = cc / a.heads, h = cc - j * a.heads;
  const int d = blockIdx.z * 128 + (tid & 31) * 4;
  bf16_t* o = a.out + (r.q0 + j) * a.o_ts + h * a.o_hs + d;
  const int tiles = (r.len + kTile - 1) / kTile;
  if (tiles == 0) {
    if (tid < 32) *reinterpret_cast<uint2*>(o) = make_uint2(0, 0);
    return;
  }
  const int per = a.starts[a.requests * a.columns16], item = a.starts[b * a.columns16 + ct];
  const int w0 = item / per, w1 = (item + tiles - 1) / per;
  if (w0 == w1) return;
  const int parts = w1 - w0 + 1;  // <= kWgs
  const int slot0 = item == w0 * per ? 2 * w0 : 2 * w0 + 1;
  float m = -__FLT_MAX__, l = 0.f;
  if (tid < parts) {
    const int slot = tid ? 2 * (w0 + tid) : slot0;
    m = a.part_ml[(slot * 16 + c) * 2];
    l = a.part_ml[(slot * 16 + c) * 2 + 1];
  }
  float mm = wave_max(m);
  if (lane == 0) red[wv] = mm;
  __syncthreads();
  mm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float w = __builtin_amdgcn_exp2f(m - mm);
  const float ls = wave_sum(l * w);
  if (lane == 0) red[4 + wv] = ls;
  wgt[tid] = w;
  __syncthreads();
  const float lsum = (red[4] + red[5]) + (red[6] + red[7]);
  const int grp = tid >> 5;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int p = grp; p < parts; p += 8) {
    const int slot = p ? 2 * (w0 + p) : slot0;
    const float4 x = *reinterpret_cast<const float4*>(a.part_o + static_cast<int64_t>(slot) * kPartFloats + c * kLat + d);
    const float f = wgt[p];
    v.x = __builtin_fmaf(f, x.x, v.x);
    v.y = __builtin_fmaf(f, x.y, v.y);
    v.z = __builtin_fmaf(f, x.z, v.z);
    v.w = __builtin_fmaf(f, x.w, v.w);
  }
  osum[grp][tid & 31] = v;
  __syncthreads();
  if (tid < 32) {
#pragma unroll
    for (int g = 1; g < 8; ++g) {
      v.x += osum[g][tid].x;
      v.y += osum[g][tid].y;
      v.z += osum[g][tid].z;
      v.w += osum[g][tid].w;
    }
    const float inv = r.len - r.nq + j + 1 > 0 ? 1.0f / lsum : 0.f;
    *reinterpret_cast<uint2*>(o) = make_uint2(pack2(v.x * inv, v.y * inv), pack2(v.z * inv, v.w * inv));
  }
}

static int column_groups(int max_q, int heads) { return (max_q * heads + 15) / 16; }

extern "C" int64_t dsv2_mla_paged_workspace_size(int requests, int max_q, int heads) {
  if (requests < 0 || max_q < 0 || heads < 0) return 0;
  const int64_t starts = static_cast<int64_t>(requests) * ((static_cast<int64_t>(max_q) * heads + 15) / 16) + 1;
  return 2 * kWgs * (kPartFloats + 32) * 4 + (starts * 4 + 15) / 16 * 16;
}

extern "C" int dsv2_mla_decode_paged_fp4(const void* q, int64_t q_ts, int64_t q_hs, int tokens, int heads,
                                         const void* pages, int64_t page_stride, int n_pages, int page_size,
                                         const int32_t* block_table, int64_t table_stride, int table_width,
                                         const int32_t* lens, int requests, const int32_t* cu_q, int max_q,
                                         float softmax_scale, void* out, int64_t out_ts, int64_t out_hs,
                                         void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  if (const int rc = paged_check_pool("mla_decode_paged_fp4", pages, page_stride, n_pages, page_size)) return rc;
  DSV2_REQUIRE(q && block_table && lens && out, DSV2_E_NULL, "mla_decode_paged_fp4: null pointer");
  DSV2_REQUIRE(tokens >= 0 && heads > 0 && heads <= 128 && requests >= 0 && requests <= kMaxRequests && max_q > 0 &&
                   max_q <= 65535 && (cu_q || requests == tokens),
               DSV2_E_SHAPE, "mla_decode_paged_fp4: bad shape (%d query tokens, %d heads, %d requests, max_q %d)", tokens,
               heads, requests, max_q);
  DSV2_REQUIRE(table_width > 0 && table_stride >= table_width, DSV2_E_SHAPE, "mla_decode_paged_fp4: block table");
  DSV2_REQUIRE(dsv2_aligned16(q) && dsv2_aligned16(out) && q_ts % 8 == 0 && q_hs % 8 == 0 && out_ts % 8 == 0 &&
                   out_hs % 8 == 0,
               DSV2_E_ALIGN, "mla_decode_paged_fp4: alignment");
  if (tokens == 0 || requests == 0) return DSV2_OK;
  if (!cu_q) max_q = 1;
  const int groups = column_groups(max_q, heads), shift = page_shift(page_size);
  const int64_t items = static_cast<int64_t>(requests) * groups;
  const int64_t room = static_cast<int64_t>(table_width) << shift;
  DSV2_REQUIRE(room <= INT32_MAX - kTile && items <= (1 << 22) && items <= INT32_MAX / ((room + kTile - 1) / kTile), DSV2_E_SHAPE,
               "mla_decode_paged_fp4: %d requests of up to %lld tokens, %d column groups each", requests, (long long)room,
               groups);
  DSV2_REQUIRE(workspace && dsv2_aligned16(workspace) &&
                   workspace_bytes >= dsv2_mla_paged_workspace_size(requests, max_q, heads),
               DSV2_E_SHAPE, "mla_decode_paged_fp4: workspace of %lld bytes", (long long)workspace_bytes);
  float* part_o = (float*)workspace;
  float* part_ml = part_o + 2 * kWgs * kPartFloats;
  int32_t* starts = (int32_t*)(part_ml + 2 * kWgs * 32);
  const PagedAttnArgs a{(const bf16_t*)q, q_ts, q_hs, tokens, heads, (const uint8_t*)pages, page_stride, n_pages,
                        shift, block_table, table_stride, table_width, lens, cu_q, max_q, requests, groups,
                        softmax_scale * 1.4426950408889634f, (bf16_t*)out, out_ts, out_hs, part_o, part_ml, starts,
                        status};
  const int64_t most = items * ((room + kTile - 1) / kTile);
  const int wgs = static_cast<int>(most / kMinTiles + 1 < kWgs ? most / kMinTiles + 1 : kWgs);
  hipLaunchKernelGGL(mla_paged_kernel, dim3(wgs), dim3(64 * kWaves), kWaves * kWaveLds + requests * 4,
                     (hipStream_t)stream, a);
  if (const int rc = dsv2_launch_status("mla_decode_paged_fp4")) return rc;
  hipLaunchKernelGGL(mla_paged_merge_kernel, dim3((unsigned)items, 16, 4), dim3(256), 0, (hipStream_t)stream, a);
  return dsv2_launch_status("mla_decode_paged_fp4");
}
