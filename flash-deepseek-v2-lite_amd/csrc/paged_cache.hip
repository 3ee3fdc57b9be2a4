// The paged latent cache: block tables and slot maps from request lengths, rows into pages and back.
#include "paged.h"

using namespace paged;

int paged_check_pool(const char* what, const void* pages, int64_t page_stride, int n_pages, int page_size) {
  DSV2_REQUIRE(pages, DSV2_E_NULL, "%s: null pages", what);
  const int shift = page_shift(page_size);
  DSV2_REQUIRE(shift >= 0, DSV2_E_SHAPE, "%s: page_size %d is no power of two in [1, 1024]", what, page_size);
  DSV2_REQUIRE(n_pages > 0 && n_pages <= (INT32_MAX >> shift), DSV2_E_SHAPE,
               "%s: %d pages of %d tokens: slots are int32", what, n_pages, page_size);
  DSV2_REQUIRE(page_stride >= static_cast<int64_t>(kTokenB) * page_size, DSV2_E_SHAPE,
               "%s: a page of %d tokens takes %d bytes", what, page_size, kTokenB * page_size);
  DSV2_REQUIRE(dsv2_aligned16(pages) && page_stride % 16 == 0, DSV2_E_ALIGN, "%s: pages alignment", what);
  return DSV2_OK;
}

// ---------------------------------------------------------------------------
// Block tables and slot maps
// ---------------------------------------------------------------------------
namespace {
constexpr int kMaxRequests = 4096;  // four int32 arrays of the requests in LDS
constexpr int kManyRequests = 512;
// sums of counts stick at the largest uint32, past every int32 that they are compared with
__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }

// first index of ends[0, n) (ascending) that is past i; i < ends[n - 1]
__device__ __forceinline__ int owner(const uint32_t* ends, int n, uint32_t i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > i)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// the sums of v[0, K) over the threads before this one, and over all; red: K words of LDS a wave
template <int K, int kWaves>
__device__ __forceinline__ void block_scan(const uint32_t* v, uint32_t* before, uint32_t* total, uint32_t* red) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto sat = [](uint32_t a, uint32_t b) { return add_sat(a, b); };
  uint32_t x[K];
#pragma unroll
  for (int k = 0; k < K; ++k) x[k] = wave_scan(v[k], sat);
  if (lane == 63) {
#pragma unroll
    for (int k = 0; k < K; ++k) red[w * K + k] = x[k];
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    before[k] = __builtin_amdgcn_update_dpp(0, x[k], 0x138, 0xf, 0xf, false);  // the lane before this one's, 0 before lane 0
  }
  __syncthreads();
  // sixteen waves' sums by a scan again (1,024 requests 8.7 -> 7.2 us), four one by one (8 requests 3.4 -> 3.25)
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (kWaves > 4) {
      const int waves = wave_scan(lane < kWaves ? red[lane * K + k] : 0u, sat);
      total[k] = __builtin_amdgcn_readlane(waves, kWaves - 1);
      if (w) before[k] = add_sat(before[k], __builtin_amdgcn_readlane(waves, w - 1));
    } else {
      total[k] = 0;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        if (i == w) before[k] = add_sat(before[k], total[k]);
        total[k] = add_sat(total[k], red[i * K + k]);
      }
    }
  }
}

struct PlanArgs {
  const int32_t* lens;   // STEP: state (lengths, then the ring's head and count); else the ranges' first tokens
  const int32_t* delta;  // STEP: change of each length; else the ranges' sizes
  int n;
  int32_t* table;
  int64_t ts;
  int width;
  int32_t* ring;
  int pages;
  int shift;
  int tokens;
  int32_t* state_out;
  int32_t* slots;
  int32_t* positions;
  int32_t* rows;
  int32_t* cu_q;  // STEP: the requests' first new tokens, or null
  int32_t* status;
};
}  // namespace

// Every workgroup scans all requests for itself (their lengths and changes are a few KB of L2 reads
// and the sums live in LDS), then takes its share of the tokens, of the pages given out and of the
// pages taken back: one launch, no workgroup waits for another, and what is read (tables below a
// request's old end, the ring's free stretch) is never what is written (entries from there on, the
// ring behind its free stretch, the new state).
//
// Request b with change d and `have` pages: d > 0 appends when its tokens fit the table's width and,
// with every earlier request's, max_tokens, and the pages needed up to it are free; the sums run over
// all requests that fit the width, so whoever is refused leaves the others' places as they were, and
// the pages given out are the ring's first ones without gaps.  d < 0 drops tokens from the end; the
// pages that empties go behind the ring's free stretch in the order of requests and pages.
//
// Integer sums, a handful of bytes: bound by the launch and a few dependent loads and barriers (MI355X, in a graph:
// 8 requests 3.3 us, of which an empty launch takes 1.7; 1,024 requests with 263,000 new tokens 7.2 us, 3.2 MB
// written; ranges of 5 requests 2.7, of 256 with 525,000 tokens 5.4 us, 6.3 MB).
template <bool STEP, int kThreads>
__global__ __launch_bounds__(kThreads) void paged_plan_kernel(const PlanArgs a) {
  constexpr int K = STEP ? 3 : 1;
  constexpr uint32_t kTaken = 0x80000000u;
  extern __shared__ uint32_t sums[];
  __shared__ uint32_t red[kThreads / 64 * K];
  __shared__ int32_t taken_sum;
  uint32_t* tok_end = sums;             // tokens of requests [0, b]
  uint32_t* page_end = sums + a.n;      // STEP: pages they need
  uint32_t* back_end = sums + 2 * a.n;  // STEP: pages they give back
  uint32_t* meta = sums + 3 * a.n;      // STEP: old length; kTaken: the new tokens fit
  const int tid = threadIdx.x;
  const int ps = 1 << a.shift;
  const int64_t room = static_cast<int64_t>(a.width) << a.shift;
  auto pages_of = [&](int64_t len) { return static_cast<uint32_t>((len + ps - 1) >> a.shift); };
  int head = 0, count = 0;
  if (STEP) {
    head = a.lens[a.n];
    count = min(max(a.lens[a.n + 1], 0), a.pages);
    head = head >= 0 && head < a.pages ? head : 0;
    if (tid == 0) taken_sum = 0;
  }
  // each thread's own run of requests, sums within the run
  const int per = (a.n + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.n), b1 = min(b0 + per, a.n);
  uint32_t run[K] = {};
  int taken = 0, errors = 0;
  for (int b = b0; b < b1; ++b) {
    const int d = a.delta[b];
    run[0] = add_sat(run[0], max(d, 0));
    tok_end[b] = run[0];
    if (STEP) {
      const int64_t len = min(max(static_cast<int64_t>(a.lens[b]), static_cast<int64_t>(0)), room);
      const int64_t want = len + d;
      const bool fits = d > 0 && want <= room;
      if (d > 0 && !fits) errors |= DSV2_DEVERR_CACHE_FULL;
      if (fits) run[1] = add_sat(run[1], pages_of(want) - pages_of(len));
      if (d < 0) run[K - 1] = add_sat(run[K - 1], pages_of(len) - pages_of(max(want, static_cast<int64_t>(0))));
      page_end[b] = run[1 % K];
      back_end[b] = run[K - 1];
      meta[b] = static_cast<uint32_t>(len) | (fits ? kTaken : 0u);
    }
  }
  uint32_t before[K], total[K];
  block_scan<K, kThreads / 64>(run, before, total, red);
  uint32_t tok_last = 0, page_last = 0;
  for (int b = b0; b < b1; ++b) {
    const uint32_t t = tok_end[b], t_end = add_sat(before[0], t);
    const bool grows = t > tok_last;
    tok_last = t;
    tok_end[b] = t_end;
    if (STEP) {
      const uint32_t p = page_end[b], p_end = add_sat(before[1 % K], p), need = p - page_last;
      page_last = p;
      page_end[b] = p_end;
      back_end[b] = add_sat(before[K - 1], back_end[b]);
      const uint32_t m = meta[b];
      const bool fits = m & kTaken;
      const bool ok = fits && t_end <= static_cast<uint32_t>(a.tokens) && (need == 0 || p_end <= static_cast<uint32_t>(count));
      if (ok) taken += need;
      if (fits && !ok) errors |= t_end > static_cast<uint32_t>(a.tokens) ? DSV2_DEVERR_TOKENS : DSV2_DEVERR_NO_PAGE;
      const int len = m & ~kTaken;
      meta[b] = ok ? m : len;
      if (blockIdx.x == 0) {
        const int d = a.delta[b];
        if (a.cu_q) a.cu_q[b + 1] = static_cast<int>(min(t_end, 0x7fffffffu));
        a.state_out[b] = d < 0 ? static_cast<int>(max(static_cast<int64_t>(len) + d, static_cast<int64_t>(0))) : (ok ? len + d : len);
      }
    } else if (t_end > static_cast<uint32_t>(a.tokens) && grows) {
      errors |= DSV2_DEVERR_TOKENS;
    }
  }
  if (STEP) {
    taken = wave_scan(taken);
    if ((tid & 63) == 63 && taken) atomicAdd(&taken_sum, taken);
  }
  __syncthreads();
  const int used = STEP ? taken_sum : 0;
  // a ring that already holds every page it could get back was not this table's: what does not fit is dropped
  const int given = STEP ? static_cast<int>(min(total[K - 1], static_cast<uint32_t>(a.pages - count))) : 0;
  if (blockIdx.x == 0) {
    if (STEP && tid == 0) {
      if (a.cu_q) a.cu_q[0] = 0;
      const int64_t h = static_cast<int64_t>(head) + used;
      a.state_out[a.n] = static_cast<int>(h >= a.pages ? h - a.pages : h);
      a.state_out[a.n + 1] = count - used + given;
      if (static_cast<uint32_t>(given) < total[K - 1]) errors |= DSV2_DEVERR_BAD_SLOT;
    }
    if (errors && a.status) atomicOr(a.status, errors);
  }

  // tokens, then (STEP) pages given out, then pages taken back, all in one line over the threads
  const int live = static_cast<int>(min(total[0], static_cast<uint32_t>(a.tokens)));
  const int64_t all = static_cast<int64_t>(a.tokens) + used + given;
  int bad = 0;
  for (int64_t at = blockIdx.x * kThreads + tid; at < all; at += gridDim.x * kThreads) {
    if (at < a.tokens) {
      const int i = static_cast<int>(at);
      int slot = -1, pos = -1, row = -1;
      if (i < live) {
        const int b = owner(tok_end, a.n, i);
        const int j = i - (b ? tok_end[b - 1] : 0);
        int page = -1;
        int64_t t = -1;
        if (STEP) {
          const uint32_t m = meta[b];
          if (m & kTaken) {
            const int have = pages_of(m & ~kTaken);
            t = static_cast<int64_t>(m & ~kTaken) + j;
            const int idx = static_cast<int>(t >> a.shift);
            if (idx < have) {
              page = a.table[b * a.ts + idx];
            } else {
              const int64_t k = static_cast<int64_t>(head) + (b ? page_end[b - 1] : 0) + idx - have;
              page = a.ring[k >= a.pages ? k - a.pages : k];
            }
            if (page >= a.pages) page = -1;
          }
        } else {
          const int s = a.lens[b];
          t = static_cast<int64_t>(s) + j;
          if (s < 0 || t >= room) {
            t = -1;
            bad = DSV2_DEVERR_BAD_SLOT;
          } else {
            page = a.table[b * a.ts + (t >> a.shift)];
            if (page > (INT32_MAX >> a.shift)) page = -1;
          }
        }
        if (t >= 0) {
          pos = static_cast<int>(t);
          row = b;
          if (page >= 0)
            slot = (page << a.shift) | (pos & (ps - 1));
          else
            bad = DSV2_DEVERR_BAD_SLOT;
        }
      }
      a.slots[i] = slot;
      a.positions[i] = pos;
      a.rows[i] = row;
    } else if (STEP && at < static_cast<int64_t>(a.tokens) + used) {
      const int k = static_cast<int>(at - a.tokens), b = owner(page_end, a.n, k);
      const int64_t r = static_cast<int64_t>(head) + k;
      a.table[b * a.ts + pages_of(meta[b] & ~kTaken) + k - (b ? page_end[b - 1] : 0)] = a.ring[r >= a.pages ? r - a.pages : r];
    } else if (STEP) {
      const int k = static_cast<int>(at - a.tokens - used), b = owner(back_end, a.n, k);
      const int first = b ? back_end[b - 1] : 0;
      const int kept = static_cast<int>(pages_of(meta[b] & ~kTaken)) - (back_end[b] - first);
      int64_t r = static_cast<int64_t>(head) + count + k;  // < 3 * pages: head, count and k are below pages each
      while (r >= a.pages) r -= a.pages;
      a.ring[r] = a.table[b * a.ts + kept + k - first];
    }
  }
  if (bad && a.status) atomicOr(a.status, bad);
}

static int plan_launch(const char* what, bool step, const PlanArgs& a, int page_size, void* stream) {
  DSV2_REQUIRE(a.n >= 0 && a.n <= kMaxRequests, DSV2_E_SHAPE, "%s: %d requests, at most %d", what, a.n, kMaxRequests);
  DSV2_REQUIRE(a.shift >= 0, DSV2_E_SHAPE, "%s: page_size %d is no power of two in [1, 1024]", what, page_size);
  DSV2_REQUIRE(a.width > 0 && a.width <= (INT32_MAX >> a.shift) && a.ts >= a.width, DSV2_E_SHAPE,
               "%s: block table of %d columns", what, a.width);
  DSV2_REQUIRE(a.tokens >= 0, DSV2_E_SHAPE, "%s: max_tokens %d", what, a.tokens);
  // Every workgroup repeats the scan, so many requests go with few, large workgroups (MI355X, us with 256 and with
  // 1,024 threads; steps whose every fourth request gains up to 2,048 tokens: 256 requests 4.7 / 4.7, 400 5.3 / 5.2, 512
  // 5.6 / 5.1, 768 6.8 / 5.7; with one token each 64 3.9 / 4.1, 512 5.6 / 5.7, 768 6.2 / 6.4; ranges of up to 2,000
  // tokens: 128 3.3 / 3.6, 512 5.6 / 5.6, 768 7.5 / 7.3, 1,024 9.8 / 8.9).  What a step takes back only the device knows:
  // room for 8 pages a request (1,000 requests, 62 of which end with 62 pages: 7.7 us, with none 10.7).
  const bool many = a.n > kManyRequests;
  const int threads = many ? 1024 : 256, most = many ? 256 : 1024;
  const int64_t all = (static_cast<int64_t>(a.tokens) + (step ? 8 : 1) * a.n + threads - 1) / threads;
  const dim3 wgs(static_cast<unsigned>(all < 1 ? 1 : (all > most ? most : all)));
  const size_t lds = static_cast<size_t>(a.n) * (step ? 16 : 4);
  hipStream_t st = (hipStream_t)stream;
  if (step && threads == 1024)
    hipLaunchKernelGGL((paged_plan_kernel<true, 1024>), wgs, dim3(1024), lds, st, a);
  else if (step)
    hipLaunchKernelGGL((paged_plan_kernel<true, 256>), wgs, dim3(256), lds, st, a);
  else if (threads == 1024)
    hipLaunchKernelGGL((paged_plan_kernel<false, 1024>), wgs, dim3(1024), lds, st, a);
  else
    hipLaunchKernelGGL((paged_plan_kernel<false, 256>), wgs, dim3(256), lds, st, a);
  return dsv2_launch_status(what);
}

extern "C" int dsv2_paged_step(const int32_t* state, const int32_t* delta, int requests, int32_t* block_table,
                               int64_t table_stride, int table_width, int32_t* free_pages, int n_pages, int page_size,
                               int max_tokens, int32_t* state_out, int32_t* slots, int32_t* positions, int32_t* rows,
                               int32_t* status, void* stream) {
  return dsv2_paged_step_queries(state, delta, requests, block_table, table_stride, table_width, free_pages, n_pages,
                                 page_size, max_tokens, state_out, slots, positions, rows, nullptr, status, stream);
}

extern "C" int dsv2_paged_step_queries(const int32_t* state, const int32_t* delta, int requests, int32_t* block_table,
                                       int64_t table_stride, int table_width, int32_t* free_pages, int n_pages,
                                       int page_size, int max_tokens, int32_t* state_out, int32_t* slots,
                                       int32_t* positions, int32_t* rows, int32_t* cu_q, int32_t* status,
                                       void* stream) {
  DSV2_REQUIRE(state && delta && block_table && free_pages && state_out && (max_tokens == 0 || (slots && positions && rows)),
               DSV2_E_NULL, "paged_step: null pointer");
  const int shift = page_shift(page_size);
  DSV2_REQUIRE(n_pages > 0 && (shift < 0 || n_pages <= (INT32_MAX >> shift)), DSV2_E_SHAPE, "paged_step: %d pages",
               n_pages);
  DSV2_REQUIRE(state_out + requests + 2 <= state || state + requests + 2 <= state_out, DSV2_E_SHAPE,
               "paged_step: state_out overlaps state");
  const PlanArgs a{state, delta, requests, block_table, table_stride, table_width, free_pages, n_pages,
                   shift, max_tokens, state_out, slots, positions, rows, cu_q, status};
  return plan_launch("paged_step", true, a, page_size, stream);
}

extern "C" int dsv2_paged_slots(const int32_t* starts, const int32_t* counts, int requests, const int32_t* block_table,
                                int64_t table_stride, int table_width, int page_size, int max_tokens, int32_t* slots,
                                int32_t* positions, int32_t* rows, int32_t* status, void* stream) {
  DSV2_REQUIRE(starts && counts && block_table && (max_tokens == 0 || (slots && positions && rows)), DSV2_E_NULL,
               "paged_slots: null pointer");
  const PlanArgs a{starts, counts, requests, const_cast<int32_t*>(block_table), table_stride, table_width, nullptr, 0,
                   page_shift(page_size), max_tokens, nullptr, slots, positions, rows, nullptr, status};
  return plan_launch("paged_slots", false, a, page_size, stream);
}

// ---------------------------------------------------------------------------
// Rows into pages and back: a wave takes a token (or R of them), a lane 8 latent values of it (4 lanes a block)
//
//   write: e = the least with max |x| <= 6 * 2^e over a block of 32, code = e2m1(x / 2^e);  read: x = code * 2^e
//
// 1,152 bytes of row and 400 of page a token, hardly an operation: bound by them, and by the launch for few rows.  A
// wave a token makes every access whole: 1,024 + 128 bytes of the row, 256 codes, 128 bytes of keys, 16 scales; the
// block's maximum stays within four lanes, two register moves.  MI355X, in a graph: 64 rows written and read back
// 4.3 us (two launches), 8,192 rows 8.6; 747 rows read 2.5 us, 65,536 16.8 (6.0 TB/s, a copy's 5.7).
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void paged_write_kernel(const bf16_t* __restrict__ rows, int64_t rs, int n,
                                                          const int32_t* __restrict__ slots,
                                                          uint8_t* __restrict__ pages, int64_t page_stride, int n_slots,
                                                          int shift, int32_t* __restrict__ status) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= n) return;
  const int slot = slots[r];
  const bf16_t* row = rows + r * rs;
  const uint4 v = ldg16(row + lane * 8);
  const uint4 k = ldg16(row + kLat + (lane & 7) * 8);
  if (slot < 0) return;
  if (slot >= n_slots) {
    if (lane == 0 && status) atomicOr(status, DSV2_DEVERR_BAD_SLOT);
    return;
  }
  // the largest magnitude of the block's 32 values, as bf16 bits (their order is that of the values,
  // infinities and NaN above all)
  uint32_t most = 0;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max(most, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
  most = max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), 0xB1, 0xF, 0xF, false)));
  most = max(most, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(most), 0x4E, 0xF, 0xF, false)));
  // 6 = 1.5 * 4: with most = 1.m * 2^E the least 2^e that holds it within 6 has e = E - 2 up to 1.5 * 2^E
  int e = static_cast<int>(most >> 7) - 129 + ((most & 0x7f) > 0x40 ? 1 : 0);
  e = min(max(e, kLeastExp), kMostExp);
  const bool odd = most >= 0x7f80u;
  const uint32_t s = odd ? kNanScale : static_cast<uint32_t>(e + 127);
  const float scale = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
  uint32_t code = 0;
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, w[0]), scale, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, w[1]), scale, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, w[2]), scale, 2);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, w[3]), scale, 3);
  const TokenAt at = token_at(slot, shift, page_stride);
  *reinterpret_cast<uint32_t*>(pages + at.code + lane * 4) = odd ? 0u : code;
  if (lane < 8) *reinterpret_cast<uint4*>(pages + at.rope + lane * 16) = k;
  if ((lane & 3) == 0) pages[at.scale + (lane >> 2)] = static_cast<uint8_t>(s);
}

// From kManyRows rows a wave reads four at once and its stores pass the caches by, below it one and plain
// stores (MI355X, us of one and of four: 1,024 rows 2.5 / 3.1, 4,096 3.2 / 3.3, 6,000 3.7 / 3.7, 8,192 4.3 / 3.8, 16,384
// 6.9 / 5.6, 65,536 23.3 / 16.8, 6.0 TB/s)
constexpr int kManyRows = 6000;

__device__ __forceinline__ void stg16_nt(void* p, const uint4& v) {
  const u32x4_t x = {v.x, v.y, v.z, v.w};
  __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t*>(p));
}

template <int R>
__global__ __launch_bounds__(256) void paged_read_kernel(const uint8_t* __restrict__ pages, int64_t page_stride,
                                                         int n_slots, int shift, const int32_t* __restrict__ slots,
                                                         int n, bf16_t* __restrict__ out, int64_t os,
                                                         int32_t* __restrict__ status) {
  const int r0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * R, lane = threadIdx.x & 63;
  if (r0 >= n) return;
  int slot[R];
#pragma unroll
  for (int i = 0; i < R; ++i) slot[i] = slots[min(r0 + i, n - 1)];
  uint32_t code[R], s[R];
  uint4 k[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    code[i] = s[i] = 0;
    k[i] = make_uint4(0, 0, 0, 0);
    if (slot[i] >= 0 && slot[i] < n_slots) {
      const TokenAt at = token_at(slot[i], shift, page_stride);
      code[i] = *reinterpret_cast<const uint32_t*>(pages + at.code + lane * 4);
      s[i] = pages[at.scale + (lane >> 2)];
      if (lane < 8) k[i] = ldg16(pages + at.rope + lane * 16);
    } else if (slot[i] >= n_slots && lane == 0 && status) {
      atomicOr(status, DSV2_DEVERR_BAD_SLOT);
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (r0 + i >= n) break;
    bf16_t* row = out + (r0 + i) * os;
    uint4 v = decode8(code[i], s[i]);
    if (s[i] == kNanScale) v = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
    if (R > 1) {
      stg16_nt(row + lane * 8, v);
      if (lane < 8) stg16_nt(row + kLat + lane * 8, k[i]);
    } else {
      *reinterpret_cast<uint4*>(row + lane * 8) = v;
      if (lane < 8) *reinterpret_cast<uint4*>(row + kLat + lane * 8) = k[i];
    }
  }
}

extern "C" int dsv2_paged_write_fp4(const void* rows, int64_t row_stride, int n, const int32_t* slots, void* pages,
                                    int64_t page_stride, int n_pages, int page_size, int32_t* status, void* stream) {
  if (const int rc = paged_check_pool("paged_write_fp4", pages, page_stride, n_pages, page_size)) return rc;
  DSV2_REQUIRE(n >= 0 && (row_stride >= kRow || row_stride == 0), DSV2_E_SHAPE, "paged_write_fp4: bad shape");
  if (n == 0) return DSV2_OK;
  DSV2_REQUIRE(rows && slots, DSV2_E_NULL, "paged_write_fp4: null pointer");
  DSV2_REQUIRE(dsv2_aligned16(rows) && row_stride % 8 == 0, DSV2_E_ALIGN, "paged_write_fp4: rows alignment");
  const int shift = page_shift(page_size);
  // a launch has fewer than 2^32 threads, 64 for a row
  constexpr int kMost = 1 << 25;
  for (int64_t first = 0; first < n; first += kMost) {
    const int some = n - first < kMost ? static_cast<int>(n - first) : kMost;
    hipLaunchKernelGGL(paged_write_kernel, dim3((some - 1) / 4 + 1), dim3(256), 0, (hipStream_t)stream,
                       (const bf16_t*)rows + first * row_stride, row_stride, some, slots + first, (uint8_t*)pages,
                       page_stride, n_pages << shift, shift, status);
    if (const int rc = dsv2_launch_status("paged_write_fp4")) return rc;
  }
  return DSV2_OK;
}

extern "C" int dsv2_paged_read_fp4(const void* pages, int64_t page_stride, int n_pages, int page_size,
                                   const int32_t* slots, int n, void* out, int64_t out_stride, int32_t* status,
                                   void* stream) {
  if (const int rc = paged_check_pool("paged_read_fp4", pages, page_stride, n_pages, page_size)) return rc;
  DSV2_REQUIRE(n >= 0 && out_stride >= kRow, DSV2_E_SHAPE, "paged_read_fp4: bad shape");
  if (n == 0) return DSV2_OK;
  DSV2_REQUIRE(slots && out, DSV2_E_NULL, "paged_read_fp4: null pointer");
  DSV2_REQUIRE(dsv2_aligned16(out) && out_stride % 8 == 0, DSV2_E_ALIGN, "paged_read_fp4: out alignment");
  const int shift = page_shift(page_size);
  if (n >= kManyRows)
    hipLaunchKernelGGL(paged_read_kernel<4>, dim3((n - 1) / 16 + 1), dim3(256), 0, (hipStream_t)stream,
                       (const uint8_t*)pages, page_stride, n_pages << shift, shift, slots, n, (bf16_t*)out, out_stride,
                       status);
  else
    hipLaunchKernelGGL(paged_read_kernel<1>, dim3((n - 1) / 4 + 1), dim3(256), 0, (hipStream_t)stream,
                       (const uint8_t*)pages, page_stride, n_pages << shift, shift, slots, n, (bf16_t*)out, out_stride,
                       status);
  return dsv2_launch_status("paged_read_fp4");
}

__global__ void paged_take_status_kernel(int32_t* bits, int32_t* status) { *bits = atomicExch(status, 0); }

extern "C" int dsv2_paged_take_status(int32_t* bits, int32_t* status, void* stream) {
  DSV2_REQUIRE(bits && status, DSV2_E_NULL, "paged_take_status: null pointer");
  hipLaunchKernelGGL(paged_take_status_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, bits, status);
  return dsv2_launch_status("paged_take_status");
}
