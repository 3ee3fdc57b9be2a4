// Absorbed-MLA attention over the paged latent cache held in 4 bits.
//
//   s_t = scale * q . (latent_t | rope_t),  p = softmax(s),  o = sum_t p_t latent_t
//
// One (query token, head) pair is a column; a request's columns are numbered token by token, and 16 of
// them make the narrow side of the MFMAs (S^T = K Q^T, O^T += V^T P^T).  An item is one request and 16 of
// its columns: ceil(length / 16) tiles of 16 tokens.
//
// Work is dealt out on the device, where the lengths are.  Items stand one after the other on a line, each
// with its tiles and kItemCost more places for what an item costs beside them (queries, the waves' joining,
// outputs); every workgroup sums the line for itself and takes an equal stretch of it.  A stretch's end
// closer than kPiece tiles to an item's end moves there, so pieces fill the waves at least once and items
// of less than two pieces are never cut.  An item within one workgroup is finished there; of one cut into
// several each leaves its part (fp32 o, max, sum) in the workspace and mla_paged_merge_kernel joins them.
//
// A token's 400 bytes give 2 * 16 * (576 + 512) operations a column group, 87 a byte: the matrix cores' rate would
// allow 200, so the pages' bytes bound it.  A wave takes a tile of 16 tokens at a time: it decodes a block of codes
// once, into registers (the K side of the scores) and into its own rows of LDS, where the outputs' products read them
// transposed (the V side); scores and outputs are fp32, the running maximum and sum stay in the wave, and the eight
// waves meet once, at a piece's end.  Splitting the outputs over the waves instead needs no such end, but its barriers
// keep the waves in step: 65.5 us where this takes 60.5.
//
// MI355X, both launches: 128 requests of 256 to 8,192 tokens, 16 heads: 60.5 us for 221 MB (3.6 TB/s; 38.8 us at the
// rate of a copy, 5.69 TB/s); the loop itself runs at that rate, some 20 us are launches (3), the first loads (4), the
// waves' meeting (5) and the merge (6).  One request of 150,000: 25.6 us; of 140: 10.5.
#include "paged.h"
#include "paged_line.h"

using namespace paged;

namespace {
constexpr int kTile = 16;
constexpr int kWaves = 8;
constexpr int kThreads = 64 * kWaves;
// LDS row of a token's latent: 1,056 bytes, with the halves of every 32 bytes swapped in rows 4-7 and
// 12-15.  Eight rows' 16-byte writes of one block then fill 128 bytes, and so do the four rows' 32 bytes
// of a transposed read
constexpr int kVRow = kLat + 16;
constexpr int kORow = kLat + 4;        // LDS row of a column's output (floats)
constexpr int kWaveLds = kTile * kVRow * 2;
constexpr int kQLds = 18 * 64 * 16;    // the item's Q^T fragments
constexpr int kQAhead = 3, kVAhead = 6;  // fragments that are read ahead of the products
constexpr int kQLoads = (18 + kWaves - 1) / kWaves;
static_assert(16 * kORow * 4 <= 2 * kWaveLds, "a wave's outputs take two tiles' place");
constexpr int kWgs = 256;              // one workgroup per CU
constexpr int kMinStretch = 2 * kPiece;
// A piece takes what some 32 more tiles would, 20,000 cycles (MI355X, 128 x 256..8,192 tokens, both launches: 62.8 us
// with 16, 60.2 with 24, 60.5 with 32, 61.7 with 40; 12 x 1,440..24,485 26.8 / 26.0 / 25.9 / 26.2)
constexpr int kItemCost = 32;
// The host refuses calls whose line would pass this (a request's columns, and all requests' by the query tokens that
// there are).  Ranges of cu_q that overlap could still add up to more: sums stop here, and no index follows from more
constexpr int kMostPlaces = 1 << 30;
__device__ __forceinline__ int add_places(int a, int b) { return min(a + b, kMostPlaces); }
constexpr int kPartFloats = 16 * kLat;
// Up to 128 requests one wave sums the line; more are shared by the workgroup (MI355X, one request, to the first item,
// each wave summing for itself: 1,850 cycles where the workgroup takes 3,400; with room for 256 requests 2,480, for 64
// some 1,700; one wave for all, which cannot part the waves, takes 0.2 us more.  By one wave / by the workgroup, us: one
// request of 140 10.6 / 10.9, 64 of 100..2,000 22.2 / 22.7, 128 28.4 / 28.5; with room for 256 requests 192 34.0 / 34.2,
// 256 41.1 / 40.6, and one request 10.9)
constexpr int kFew = 2;

struct PagedAttnArgs {
  const bf16_t* q;
  int64_t q_ts, q_hs;
  int tokens, heads;
  uint32_t heads_inv;  // ceil(2^32 / heads), 0 for one head
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
  float scale_log2;
  bf16_t* out;
  int64_t o_ts, o_hs;
  float* part_o;     // [2 * kWgs][16][512]
  float* part_ml;    // [2 * kWgs][16][2]
  int4* cuts;        // [kWgs][2]: the item that a workgroup's first piece continues (first column or -1, its
                     // request's columns, the workgroups that it begins and ends in) and its request
  int32_t* status;
};

// column / heads: exact for columns below 2^25 and up to 128 heads (the product is less than column / 2^32 * 128 above
// the quotient times 2^32); a division by a run-time value takes some 40 instructions
__device__ __forceinline__ int token_of(const PagedAttnArgs& a, int column) {
  return a.heads_inv ? static_cast<int>(__umulhi(static_cast<uint32_t>(column), a.heads_inv)) : column;
}
// n / d for 0 <= n < 2^20, d > 0: (n + 1/2) / d is 1 / (2 d) from the next whole number, its error below (n + 1/2) / d / 2^22
__device__ __forceinline__ int quotient(int n, int d) {
  return static_cast<int>((static_cast<float>(n) + 0.5f) * __builtin_amdgcn_rcpf(static_cast<float>(d)));
}
// the output row of a column of the request whose first query token is q0
__device__ __forceinline__ bf16_t* out_row(const PagedAttnArgs& a, int q0, int column) {
  const int j = token_of(a, column);
  return a.out + (q0 + j) * a.o_ts + (column - j * a.heads) * a.o_hs;
}

// a value that all lanes have, to scalar registers: what follows from it stays off the vector units
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

struct Request {
  int len, q0, nq, columns;
  __device__ __forceinline__ int tiles() const { return (len + kTile - 1) / kTile; }
  // its places on the line of all items
  __device__ __forceinline__ int places() const {
    return len > 0 ? (tiles() + kItemCost) * ((columns + 15) / 16) : 0;
  }
};
__device__ __forceinline__ Request uniform(const Request& r) {
  return {uniform(r.len), uniform(r.q0), uniform(r.nq), uniform(r.columns)};
}
__device__ __forceinline__ Request of_lane(const Request& r, int lane) {
  return {__builtin_amdgcn_readlane(r.len, lane), __builtin_amdgcn_readlane(r.q0, lane),
          __builtin_amdgcn_readlane(r.nq, lane), __builtin_amdgcn_readlane(r.columns, lane)};
}
__device__ __forceinline__ Request request(const PagedAttnArgs& a, int b) {
  Request r;
  const int len = a.lens[b];
  r.q0 = b;
  int end = b + 1;
  if (a.cu_q) {
    r.q0 = a.cu_q[b];
    end = a.cu_q[b + 1];
    pin(end);  // all three are requested before the first is waited for
  }
  r.len = min(max(len, 0), a.width << a.shift);  // the host has checked that this is an int32
  r.nq = r.q0 >= 0 ? max(min(end, a.tokens) - r.q0, 0) : 0;
  r.columns = min(r.nq, a.max_q) * a.heads;
  return r;
}

// a tile's bytes: lane (li, kg) has token li's latent blocks 4c + kg (32 codes each), its 16 scales and
// its rotary keys y * 32 + kg * 8 .. +8
struct Raw {
  uint4 code[4];
  uint4 rope[2];
  uint4 scale;
  bool ok;  // the token exists and its page is one
};

__device__ __forceinline__ floatx4_t mfma16x16x16(const uint2& a, const uint2& b, const floatx4_t& c) {
  typedef short short4_t __attribute__((ext_vector_type(4)));
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4_t, a), __builtin_bit_cast(short4_t, b), c, 0, 0, 0);
}
}  // namespace

// kOnePage (pages of at least a tile, whose tiles then lie in one page each): a tile's address is the wave's, in
// scalar registers, and the lanes' offsets never change; with smaller pages every lane has its own
template <bool kOnePage>
__global__ __launch_bounds__(kThreads, 2) void mla_paged_kernel(const PagedAttnArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  __shared__ float ml[kWaves][16][2];
  __shared__ int32_t wave_sums[kWaves];
  // what one wave or thread has found for all, so that the waves never part, whatever another stream does to the
  // lengths meanwhile: a request, in turns (place on the line; itself)
  __shared__ int4 found[2][2];
  uint4* const q_lds = reinterpret_cast<uint4*>(smem + kWaves * kWaveLds);
  const int tid = threadIdx.x, lane = tid & 63, wv = uniform(tid >> 6), li = lane & 15,
            kg = lane >> 4;

  // the length of the line (the host has checked that it stays within int32), and the request that this
  // workgroup's stretch begins in
  int lo, hi, per, b, start;
  Request r;
  {
    auto seen = [&](const Request& r) {
      if (r.nq > a.max_q && blockIdx.x == 0 && a.status) atomicOr(a.status, DSV2_DEVERR_TOKENS);
      return r.len == 0 && r.columns > 0;
    };
    // requests with nothing cached: zeros
    auto clear = [&] {
      for (int i = blockIdx.x; i < a.requests; i += gridDim.x) {
        const Request z = request(a, i);
        if (z.len > 0) continue;
        for (int f = tid; f < z.columns * (kLat / 8); f += kThreads) {
          *reinterpret_cast<uint4*>(out_row(a, z.q0, f / (kLat / 8)) + f % (kLat / 8) * 8) = make_uint4(0, 0, 0, 0);
        }
      }
    };
    // this workgroup's stretch of the line; none: lo == hi == total
    auto stretch = [&](int total) {
      per = max((total + kWgs - 1) / kWgs, kMinStretch);
      const int64_t from = static_cast<int64_t>(blockIdx.x) * per;
      lo = static_cast<int>(min(from, static_cast<int64_t>(total)));
      hi = min(lo + per, total);
    };
    if (tid == 0) a.cuts[2 * blockIdx.x] = make_int4(-1, 0, 0, 0);
    if (a.requests <= kFew * 64) {
      // one wave: lane l has requests l, l + 64, ...
      if (wv == 0) {
        Request u[kFew];
        int run[kFew], scan[kFew], total = 0;
        bool nothing = false;
#pragma unroll
        for (int k = 0; k < kFew; ++k) u[k] = request(a, min(64 * k + lane, a.requests - 1));
#pragma unroll
        for (int k = 0; k < kFew; ++k) {
          const bool is = 64 * k + lane < a.requests;
          nothing |= is && seen(u[k]);
          run[k] = is ? u[k].places() : 0;
          scan[k] = add_places(wave_scan(run[k], add_places), total);
          total = __builtin_amdgcn_readlane(scan[k], 63);
        }
        stretch(total);
        const bool none = __any(nothing);
        if (lane == 0) found[0][0] = make_int4(0, 0, total, none);
#pragma unroll
        for (int k = 0; k < kFew; ++k) {
          if (scan[k] - run[k] <= lo && lo < scan[k]) {
            found[0][0] = make_int4(64 * k + lane, scan[k] - run[k], total, none);
            found[0][1] = make_int4(u[k].len, u[k].q0, u[k].nq, u[k].columns);
          }
        }
      }
      __syncthreads();
      if (found[0][0].w) clear();
      stretch(uniform(found[0][0].z));
    } else {
      const int chunk = (a.requests + kThreads - 1) / kThreads;
      const int b0 = min(tid * chunk, a.requests), b1 = min(b0 + chunk, a.requests);
      int run = 0;
      bool nothing = false;
      for (int i = b0; i < b1; ++i) {
        r = request(a, i);
        nothing |= seen(r);
        run = add_places(run, r.places());
      }
      const int scan = wave_scan(run, add_places);
      if (lane == 63) wave_sums[wv] = scan;
      if (__syncthreads_or(nothing)) clear();
      int before = scan - run, total = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        if (i < wv) before = add_places(before, wave_sums[i]);
        total = add_places(total, wave_sums[i]);
      }
      stretch(uniform(total));
      if (before <= lo && lo < before + run) {
        int i = b0;
        if (b1 - b0 > 1)
          for (;; ++i) {
            r = request(a, i);
            if (i + 1 == b1 || lo < before + r.places()) break;
            before += r.places();
          }
        found[0][0] = make_int4(i, before, 0, 0);
        found[0][1] = make_int4(r.len, r.q0, r.nq, r.columns);
      }
      __syncthreads();
    }
    if (lo >= hi) return;
    const int4 u = found[0][0], v = found[0][1];
    b = uniform(u.x);
    start = uniform(u.y);
    r = uniform(Request{v.x, v.y, v.z, v.w});
  }

  bf16_t* const vt = reinterpret_cast<bf16_t*>(smem + wv * kWaveLds);
  int ct = 0;
  if (r.columns > 16) {
    ct = (lo - start) / (r.tiles() + kItemCost);
    start += ct * (r.tiles() + kItemCost);  // of the item
  }
  bool again = false;
  int turn = 0;
  for (; start < hi; start += r.tiles() + kItemCost, ++ct) {
    if (ct * 16 >= r.columns) {
      // the next request that has places (there is one, the line goes on), looked for 64 at a time: of a server's
      // rows most may be idle (8 of 4,096 in use: 71 us one after the other, 33 so)
      turn ^= 1;
      if (wv == 0) {
        uint64_t has = 0;
        for (++b; b < a.requests; b += 64) {
          r = request(a, min(b + lane, a.requests - 1));
          has = __ballot(b + lane < a.requests && r.places() > 0);
          if (has) break;
        }
        if (has ? lane == __builtin_ctzll(has) : lane == 0) {
          found[turn][0] = make_int4(has ? b + lane : -1, 0, 0, 0);
          found[turn][1] = make_int4(r.len, r.q0, r.nq, r.columns);
        }
      }
      __syncthreads();
      const int4 v = found[turn][1];
      b = uniform(found[turn][0].x);
      if (b < 0) return;
      r = uniform(Request{v.x, v.y, v.z, v.w});
      ct = 0;
    }
    // (the compiler does not see that these are the same for all lanes)
    r = uniform(r);
    b = uniform(b);
    ct = uniform(ct);
    start = uniform(start);
    const int tiles = r.tiles();
    const int t_first = cut_at(lo - start, tiles), t_last = cut_at(hi - start, tiles);
    if (t_first >= t_last) continue;
    if (again) __syncthreads();  // the last item's outputs, queries and maxima lay where this one's go
    again = true;

    const int cc = ct * 16 + li, token = token_of(a, cc);
    const int seen = cc < r.columns ? max(r.len - r.nq + token + 1, 0) : 0;

    const int32_t* row = a.table + b * a.ts;
    const int end = t_last - 1;
    auto load_page = [&](int tile) {
      const int t = min(tile, end) * kTile;
      return row[(kOnePage ? t : min(t + li, r.len - 1)) >> a.shift];
    };
    // past the last tile nothing is read: with one page a tile by a buffer of no bytes (a branch around the loads
    // would make the compiler wait for them in it), else the last tile again
    auto load_tile = [&](int tile, int pg, Raw& w) {
      const int t0 = min(tile, end) * kTile;
      if (kOnePage) pg = uniform(pg);
      const bool page = pg >= 0 && pg < a.n_pages;
      const int t = kOnePage ? t0 : min(t0 + li, r.len - 1);
      w.ok = page && t0 + li < r.len;
      if (!page && kg == 0 && t0 + li < r.len && a.status) atomicOr(a.status, DSV2_DEVERR_BAD_SLOT);
      const int off = t & ((1 << a.shift) - 1);
      const uint8_t* base = a.pages + (page ? pg : 0) * a.page_stride;
      if (kOnePage) {
        const auto buf = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0,
                                                           tile < t_last ? kTokenB << a.shift : 0, 0x27000);
        auto load = [&](int lane_at, int at) {
          return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(buf, lane_at, at, 0));
        };
#pragma unroll
        for (int c = 0; c < 4; ++c) w.code[c] = load(li * kCodeB + kg * 16 + c * 64, off * kCodeB);
#pragma unroll
        for (int y = 0; y < 2; ++y) w.rope[y] = load(li * kRopeB + kg * 16 + y * 64, (kCodeB << a.shift) + off * kRopeB);
        w.scale = load(li * kScaleB, ((kCodeB + kRopeB) << a.shift) + off * kScaleB);
      } else {
        const uint8_t *code = base + off * kCodeB, *rope = base + (kCodeB << a.shift) + off * kRopeB;
#pragma unroll
        for (int c = 0; c < 4; ++c) w.code[c] = ldg16(code + kg * 16 + c * 64);
#pragma unroll
        for (int y = 0; y < 2; ++y) w.rope[y] = ldg16(rope + kg * 16 + y * 64);
        w.scale = ldg16(base + ((kCodeB + kRopeB) << a.shift) + off * kScaleB);
      }
    };

    float m_run = -__FLT_MAX__, l_run = 0.f;
    floatx4_t acc[32];

    auto tile_step = [&](int tile, Raw& w) {
      uint32_t s[4];
      const uint32_t sw[4] = {w.scale.x, w.scale.y, w.scale.z, w.scale.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) s[c] = (sw[c] >> (8 * kg)) & 0xff;
      // rare: a token past the end or on no page (zeros), a block of NaN (its codes are zeros; one rotary
      // key becomes NaN instead, so that only the queries that see the token get NaN: a NaN latent times
      // an unseen token's p = 0 would be one too)
      const bool nan = max(max(s[0], s[1]), max(s[2], s[3])) == kNanScale;
      if (__any(!w.ok || nan)) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          w.code[c] = keep_if(w.ok && s[c] != kNanScale, w.code[c]);
          s[c] = w.ok && s[c] != kNanScale ? s[c] : 127;
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) w.rope[y] = keep_if(w.ok, w.rope[y]);
        if (nan && w.ok) w.rope[0].x = 0x7fc07fc0u;
      }
      floatx4_t sc = floatx4_t{0.f, 0.f, 0.f, 0.f};
      // three Q fragments ahead (below: six V^T fragments): left to itself the compiler reads each into the same
      // registers and waits for it (128 x 256..8,192 tokens, both launches: 65.8 -> 61.3 us)
      uint4 qa[kQAhead];
#pragma unroll
      for (int i = 0; i < kQAhead; ++i) qa[i] = q_lds[i * 64 + lane];
      bf16_t* vr = vt + li * kVRow + kg * 32;
      const int swap = (li & 4) * 2;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t cw[4] = {w.code[c].x, w.code[c].y, w.code[c].z, w.code[c].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint4 v = decode8(cw[x], s[c]);
          *reinterpret_cast<uint4*>(vr + c * 128 + ((x * 8) ^ swap)) = v;
          const int i = c * 4 + x;
          sc = mfma16x16x32(as_bf16x8(v), as_bf16x8(qa[i % kQAhead]), sc);
          if (i + kQAhead < 18) qa[i % kQAhead] = q_lds[(i + kQAhead) * 64 + lane];
        }
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) sc = mfma16x16x32(as_bf16x8(w.rope[y]), as_bf16x8(qa[(16 + y) % kQAhead]), sc);
      __builtin_amdgcn_sched_group_barrier(0x100, kQAhead, 0);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
        __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if (i + kQAhead < 18) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
      asm volatile("" ::: "memory");
      float p[4], mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = tile * kTile + 4 * kg + i < seen ? sc[i] : -INFINITY;
        mx = fmaxf(mx, p[i]);
      }
      mx = xor32_max(xor16_max(mx));
      // lazy rescaling: the running maximum (a score, not scaled yet) moves, and o and l are rescaled, only where a
      // tile exceeds it by more than 8 in log2 units, so p <= 256; it starts below every finite score.  Differences
      // are scaled, not scores: those are exact next to the maximum, however large the scores are or become when scaled
      const bool grow = (mx - m_run) * a.scale_log2 > 8.f;
      if (__any(grow)) {
        const float m_new = grow ? mx : m_run;
        const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * a.scale_log2);
        l_run *= alpha;
        m_run = m_new;
#pragma unroll
        for (int f = 0; f < 32; ++f) acc[f] *= alpha;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f((p[i] - m_run) * a.scale_log2);
      // P^T (B operand): column li, tokens 4 kg + e; the V^T fragments take the same tokens through
      // transposed reads (lane (li, kg) addresses token 4 kg + li / 4).  p is rounded to bf16, which the products take
      // (2^-8 of a weight at most), and l sums the rounded values in fp32, so the weights add up to one: a token that
      // stands alone comes out as it is held.  With p as the sum of two bf16 instead, whose products take the other
      // half of the wider MFMA's K, the errors against 64 bits are 0.00166 for 0.00176 and 128 x 256..8,192 tokens
      // take 63.6 us for 60.8, with four queries a request 49.0 for 45.0 (64 x 1,024..4,096)
      const uint2 pb = make_uint2(pack2(p[0], p[1]), pack2(p[2], p[3]));
      l_run += (__uint_as_float(pb.x << 16) + __uint_as_float(pb.x & 0xffff0000u)) +
               (__uint_as_float(pb.y << 16) + __uint_as_float(pb.y & 0xffff0000u));  // the lanes meet at the end
      const bf16_t* vp = vt + (4 * kg + (li >> 2)) * kVRow + ((4 * (li & 3)) ^ ((kg & 1) * 8));
      uint2 va[kVAhead];
#pragma unroll
      for (int f = 0; f < kVAhead; ++f) va[f] = lds_read_tr16(vp + f * 16);
#pragma unroll
      for (int f = 0; f < 32; ++f) {
        acc[f] = mfma16x16x16(va[f % kVAhead], pb, acc[f]);
        if (f + kVAhead < 32) va[f % kVAhead] = lds_read_tr16(vp + (f + kVAhead) * 16);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, kVAhead, 0);
#pragma unroll
      for (int f = 0; f < 32 - kVAhead; ++f) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, kVAhead, 0);
      asm volatile("" ::: "memory");
    };

    // wave w takes tiles t_first + w, + 8, ...: one ahead in registers, its page number one further
    {
      int tile = t_first + wv;
      Raw w0, w1;
      int pg = load_page(tile);
      // Q^T fragments (B operand), once for all waves; the k order of a block group's four products is the
      // lanes' own: k-slot (kg, e) of product (c, x) is latent (4c + kg) * 32 + x * 8 + e
      uint4 qf[kQLoads];
      const int cq = min(cc, r.columns - 1), tq = token_of(a, cq);
      const bf16_t* qrow = a.q + (r.q0 + tq) * a.q_ts + (cq - tq * a.heads) * a.q_hs;
#pragma unroll
      for (int n = 0; n < kQLoads; ++n) {
        const int i = min(wv + n * kWaves, 17);
        const int dim = i < 16 ? ((i >> 2) * 4 + kg) * 32 + (i & 3) * 8 : kLat + (i - 16) * 32 + kg * 8;
        qf[n] = ldg16(qrow + dim);
      }
      load_tile(tile, pg, w0);
      pg = load_page(tile + kWaves);
#pragma unroll
      for (int f = 0; f < 32; ++f) {
        acc[f] = floatx4_t{0.f, 0.f, 0.f, 0.f};
        asm volatile("" : "+v"(acc[f]));
      }
#pragma unroll
      for (int n = 0; n < kQLoads; ++n) {
        const int i = wv + n * kWaves;
        if (i < 18) q_lds[i * 64 + lane] = keep_if(cc < r.columns, qf[n]);
      }
      __syncthreads();  // Q
#pragma unroll 1
      for (; tile < t_last; tile += kWaves) {
        const int pn = load_page(tile + 2 * kWaves);
        load_tile(tile + kWaves, pg, w1);
        pg = pn;
        tile_step(tile, w0);
        w0 = w1;
      }
    }
    l_run = xor32_sum(xor16_sum(l_run));

    // the waves' parts meet in LDS, in the tiles' place: the upper four's, then the sums of pairs
    if (kg == 0) {
      ml[wv][li][0] = m_run;
      ml[wv][li][1] = l_run;
    }
    __syncthreads();
    float m_all = -__FLT_MAX__, l_all = 0.f, part[kWaves];
#pragma unroll
    for (int i = 0; i < kWaves; ++i) m_all = fmaxf(m_all, part[i] = ml[i][li][0]);
#pragma unroll
    for (int i = 0; i < kWaves; ++i) l_all += ml[i][li][1] * __builtin_amdgcn_exp2f((part[i] - m_all) * a.scale_log2);
    const bool whole = t_first == 0 && t_last == tiles;
    float weight = __builtin_amdgcn_exp2f((m_run - m_all) * a.scale_log2);
    if (whole) weight *= seen > 0 ? 1.0f / l_all : 0.f;
    float* o_lds = reinterpret_cast<float*>(smem + (wv & 3) * 2 * kWaveLds) + li * kORow + 4 * kg;
    if (wv >= 4) {
#pragma unroll
      for (int f = 0; f < 32; ++f) {
        const floatx4_t v = acc[f] * weight;
        *reinterpret_cast<float4*>(o_lds + f * 16) = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    __syncthreads();
    if (wv < 4) {
#pragma unroll
      for (int f = 0; f < 32; ++f) {
        const float4 u = *reinterpret_cast<const float4*>(o_lds + f * 16);
        const floatx4_t v = acc[f] * weight;
        *reinterpret_cast<float4*>(o_lds + f * 16) = make_float4(v[0] + u.x, v[1] + u.y, v[2] + u.z, v[3] + u.w);
      }
    }
    __syncthreads();
    const int slot = 2 * blockIdx.x + (t_first == 0);
    if (t_first > 0 && tid == 0) {
      int by = per;
      asm volatile("" : "+s"(by));  // the divisions are only done here
      const Parts parts = parts_of(start, tiles, by, gridDim.x);
      a.cuts[2 * blockIdx.x] = make_int4(ct * 16, r.columns, parts.first, parts.last);
      a.cuts[2 * blockIdx.x + 1] = make_int4(r.len, r.nq, r.q0, 0);
    }
#pragma unroll 1
    for (int i = 0; i < kPartFloats / 4 / kThreads; ++i) {
      const int f = tid + kThreads * i, c = f >> 7, d = (f & 127) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float4 x =
            *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + u * 2 * kWaveLds) + c * kORow + d);
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
      *reinterpret_cast<uint2*>(out_row(a, r.q0, cc) + d) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
    }
    if (!whole && tid < 16) *reinterpret_cast<float2*>(a.part_ml + (slot * 16 + tid) * 2) = make_float2(m_all, l_all);
  }
}

// Joins the parts of items that were cut.  Workgroup x stands for the cut between workgroups x and x + 1 of
// the first launch: an item in n parts has n - 1 of them, which share its 16 x 512 outputs, so each reads
// some 32 KB for each part more than one, however the parts are spread over items.  Everything that it needs
// is requested at once, when it knows its item: a thread's part of the outputs takes 8 loads at most (2 and 4
// parts: 4 and 2 times all parts; 8: 8 parts; 256: every 56th part of 9 groups of four outputs, 5 loads).
// Bound by two loads that wait for one another (cuts; maxima, sums and parts) and its launch: 5.3 us on MI355X for 255
// cuts of one item, 5.8 for some 200 of 128.  Joining in the workgroup that ends last would save the
// launch, but needs counters that are zero at each call's start, which two captured graphs would share.
__global__ __launch_bounds__(512) void mla_paged_merge_kernel(const PagedAttnArgs a) {
  constexpr int kLoads = 8, kLaneParts = kWgs / 64;
  __shared__ float weight[16][kWgs];   // of column (relative to the share's first) and part
  __shared__ float4 sums[512];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int4 item = a.cuts[2 * (blockIdx.x + 1)], req = a.cuts[2 * (blockIdx.x + 1) + 1];
  if (item.x < 0) return;
  const int col0 = item.x, columns = item.y, w0 = item.z, parts = item.w - w0 + 1;  // 2 .. kWgs
  const int share = quotient(kPartFloats / 4 + parts - 2, parts - 1);  // groups of four outputs
  const int f0 = (blockIdx.x - w0) * share, f1 = min(f0 + share, kPartFloats / 4);
  if (f0 >= f1) return;
  const int c0 = f0 >> 7, c1 = (f1 - 1) >> 7;
  auto slot = [&](int p) { return 2 * (w0 + p) + (p == 0); };
  float2 ml[2][kLaneParts];  // wave w: columns c0 + w and c0 + w + 8, lane l: parts l, l + 64, ...
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < kLaneParts; ++k) {
      const int c = c0 + wv + 8 * i, p = lane + 64 * k;
      ml[i][k] = make_float2(-__FLT_MAX__, 0.f);
      if (c <= c1 && p < parts) ml[i][k] = *reinterpret_cast<const float2*>(a.part_ml + (slot(p) * 16 + c) * 2);
    }
  // threads in groups of the share's width, each group every so many parts; a share wider than the
  // workgroup goes in passes
  const int width = min(f1 - f0, 512), groups = quotient(512, width), g = quotient(tid, width);
  const int in_pass = quotient(parts + groups - 1, groups), loads = quotient(f1 - f0 + width - 1, width) * in_pass;
  float4 x[kLoads];
  int f = f0 + tid - g * width, p = g, pass = 0;  // of the next load
  auto advance = [&] {
    p += groups;
    if (++pass < in_pass) return false;
    pass = 0;
    p = g;
    f += width;
    return true;
  };
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (k < loads && g < groups && f < f1 && p < parts)
      x[k] = *reinterpret_cast<const float4*>(a.part_o + static_cast<int64_t>(slot(p)) * kPartFloats + f * 4);
    advance();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = c0 + wv + 8 * i;
    if (c > c1) break;
    float m = ml[i][0].x;
#pragma unroll
    for (int k = 1; k < kLaneParts; ++k) m = fmaxf(m, ml[i][k].x);
    m = wave_max(m);
    float l = 0.f, w[kLaneParts];
#pragma unroll
    for (int k = 0; k < kLaneParts; ++k) {
      w[k] = __builtin_amdgcn_exp2f((ml[i][k].x - m) * a.scale_log2);
      l += ml[i][k].y * w[k];
    }
    l = wave_sum(l);
    const int cc = col0 + c;
    const float inv = cc < columns && req.x - req.y + token_of(a, cc) + 1 > 0 ? 1.0f / l : 0.f;
#pragma unroll
    for (int k = 0; k < kLaneParts; ++k)
      if (lane + 64 * k < parts) weight[c - c0][lane + 64 * k] = w[k] * inv;
  }
  __syncthreads();
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  f = f0 + tid - g * width;
  p = g;
  pass = 0;
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    if (k >= loads) break;
    const int at = f, c = at >> 7;
    if (g < groups && at < f1 && p < parts) {
      const float w = weight[c - c0][p];
      v.x = __builtin_fmaf(w, x[k].x, v.x);
      v.y = __builtin_fmaf(w, x[k].y, v.y);
      v.z = __builtin_fmaf(w, x[k].z, v.z);
      v.w = __builtin_fmaf(w, x[k].w, v.w);
    }
    if (!advance()) continue;
    if (groups > 1) {  // one pass: the groups' sums by eights, then those
      auto add = [&](int from, int by) {
        for (int i = from; i < groups; i += by) {
          const float4 u = sums[i * width + tid - g * width];
          v.x += u.x;
          v.y += u.y;
          v.z += u.z;
          v.w += u.w;
        }
      };
      sums[tid] = v;
      __syncthreads();
      if (g < 8) add(g + 8, 8);
      __syncthreads();
      if (g < 8) sums[tid] = v;
      __syncthreads();
      if (g == 0) {
        for (int i = 1; i < min(groups, 8); ++i) {
          const float4 u = sums[i * width + tid];
          v.x += u.x;
          v.y += u.y;
          v.z += u.z;
          v.w += u.w;
        }
      }
    }
    const int cc = col0 + c;
    if (g == 0 && at < f1 && cc < columns)
      *reinterpret_cast<uint2*>(out_row(a, req.z, cc) + (at & 127) * 4) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
    v = make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

extern "C" int64_t dsv2_mla_paged_workspace_size(void) {
  return kWgs * (2 * (kPartFloats + 32) * 4 + 32);
}

extern "C" int dsv2_mla_decode_paged_fp4(const void* q, int64_t q_ts, int64_t q_hs, int tokens, int heads,
                                         const void* pages, int64_t page_stride, int n_pages, int page_size,
                                         const int32_t* block_table, int64_t table_stride, int table_width,
                                         const int32_t* lens, int requests, const int32_t* cu_q, int max_q,
                                         float softmax_scale, void* out, int64_t out_ts, int64_t out_hs,
                                         void* workspace, int64_t workspace_bytes, int32_t* status, void* stream) {
  if (const int rc = paged_check_pool("mla_decode_paged_fp4", pages, page_stride, n_pages, page_size)) return rc;
  DSV2_REQUIRE(q && block_table && lens && out, DSV2_E_NULL, "mla_decode_paged_fp4: null pointer");
  DSV2_REQUIRE(tokens >= 0 && heads > 0 && heads <= 128 && requests >= 0 && requests <= 65535 && max_q > 0 &&
                   max_q <= 65535 && (cu_q || requests == tokens),
               DSV2_E_SHAPE, "mla_decode_paged_fp4: bad shape (%d query tokens, %d heads, %d requests, max_q %d)", tokens,
               heads, requests, max_q);
  DSV2_REQUIRE(table_width > 0 && table_stride >= table_width, DSV2_E_SHAPE, "mla_decode_paged_fp4: block table");
  // the largest product is the largest score only then; zero or an infinity would make masked scores NaN
  DSV2_REQUIRE(softmax_scale > 0.f && softmax_scale <= 1e30f, DSV2_E_SHAPE,
               "mla_decode_paged_fp4: softmax_scale %g is not in (0, 1e30]", softmax_scale);
  DSV2_REQUIRE(dsv2_aligned16(q) && dsv2_aligned16(out) && q_ts % 8 == 0 && q_hs % 8 == 0 && out_ts % 8 == 0 &&
                   out_hs % 8 == 0,
               DSV2_E_ALIGN, "mla_decode_paged_fp4: alignment");
  if (tokens == 0 || requests == 0) return DSV2_OK;
  if (!cu_q) max_q = 1;
  // column groups of a request and of all: no more than the query tokens have, one a request rounded up
  const int groups = ((max_q < tokens ? max_q : tokens) * heads + 15) / 16, shift = page_shift(page_size);
  const int64_t by_request = static_cast<int64_t>(requests) * groups;
  const int64_t by_token = static_cast<int64_t>(tokens) * heads / 16 + requests;
  const int64_t items = by_request < by_token ? by_request : by_token;
  const int64_t room = static_cast<int64_t>(table_width) << shift;
  DSV2_REQUIRE(room <= INT32_MAX - kTile && items <= kMostPlaces / ((room + kTile - 1) / kTile + kItemCost), DSV2_E_SHAPE,
               "mla_decode_paged_fp4: %lld groups of 16 (query token, head) pairs over up to %lld tokens each",
               (long long)items, (long long)room);
  DSV2_REQUIRE(workspace && dsv2_aligned16(workspace) &&
                   workspace_bytes >= dsv2_mla_paged_workspace_size(),
               DSV2_E_SHAPE, "mla_decode_paged_fp4: workspace of %lld bytes", (long long)workspace_bytes);
  float* part_o = (float*)workspace;
  float* part_ml = part_o + 2 * kWgs * kPartFloats;
  int4* cuts = (int4*)(part_ml + 2 * kWgs * 32);
  const PagedAttnArgs a{(const bf16_t*)q, q_ts, q_hs, tokens, heads,
                        heads == 1 ? 0u : static_cast<uint32_t>(((1ull << 32) + heads - 1) / heads),
                        (const uint8_t*)pages, page_stride, n_pages, shift, block_table, table_stride,
                        table_width, lens, cu_q, max_q, requests, softmax_scale * 1.4426950408889634f, (bf16_t*)out, out_ts,
                        out_hs, part_o, part_ml, cuts, status};
  const int64_t tiles = (room + kTile - 1) / kTile, most = items * (tiles + kItemCost);
  const int wgs = static_cast<int>(most / kMinStretch + 1 < kWgs ? most / kMinStretch + 1 : kWgs);
  constexpr int kLds = kWaves * kWaveLds + kQLds;
  if (page_size >= kTile)
    hipLaunchKernelGGL(mla_paged_kernel<true>, dim3(wgs), dim3(kThreads), kLds, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(mla_paged_kernel<false>, dim3(wgs), dim3(kThreads), kLds, (hipStream_t)stream, a);
  if (const int rc = dsv2_launch_status("mla_decode_paged_fp4")) return rc;
  if (wgs == 1 || tiles < 2 * kPiece) return DSV2_OK;  // no item of so few tiles is cut
  hipLaunchKernelGGL(mla_paged_merge_kernel, dim3(wgs - 1), dim3(512), 0, (hipStream_t)stream, a);
  return dsv2_launch_status("mla_decode_paged_fp4");
}
