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
constexpr int kPlanWgs = 512;

__device__ __forceinline__ int clamp32(int64_t v) { return static_cast<int>(min(v, static_cast<int64_t>(INT32_MAX))); }

// first index of ends[0, n) (ascending) that is past i; i < ends[n - 1]
__device__ __forceinline__ int owner(const int32_t* ends, int n, int i) {
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

// inclusive prefix sums of v over the 256 threads, and the total; red: 4 int64 of LDS
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* red, int64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(static_cast<long long>(v), o, DSV2_WAVE);
    if (lane >= o) v += u;
  }
  if (lane == 63) red[w] = v;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < w) before += red[i];
    total += red[i];
  }
  __syncthreads();
  return v + before;
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
template <bool STEP>
__global__ __launch_bounds__(256) void paged_plan_kernel(const PlanArgs a) {
  extern __shared__ int32_t sums[];
  __shared__ int64_t red[4];
  __shared__ int32_t taken_sum;
  int32_t* tok_end = sums;              // tokens of requests [0, b]
  int32_t* page_end = sums + a.n;       // STEP: pages they need
  int32_t* back_end = sums + 2 * a.n;   // STEP: pages they give back
  uint32_t* meta = reinterpret_cast<uint32_t*>(sums + 3 * a.n);  // STEP: old length, bit 31: the tokens were taken
  const int tid = threadIdx.x;
  const int ps = 1 << a.shift;
  const int64_t room = static_cast<int64_t>(a.width) << a.shift;
  int head = 0, count = 0;
  if (STEP) {
    head = a.lens[a.n];
    count = min(max(a.lens[a.n + 1], 0), a.pages);
    head = head >= 0 && head < a.pages ? head : 0;
    if (tid == 0) taken_sum = 0;
  }
  const int per = (a.n + 255) / 256;
  const int b0 = min(tid * per, a.n), b1 = min(b0 + per, a.n);
  int64_t tok = 0, page = 0, back = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t d = a.delta[b];
    tok += max(d, static_cast<int64_t>(0));
    tok_end[b] = clamp32(tok);  // within the thread's own run for now
    if (STEP) {
      const int64_t len = min(max(static_cast<int64_t>(a.lens[b]), static_cast<int64_t>(0)), room);
      const int64_t want = len + d;
      const int64_t have = (len + ps - 1) >> a.shift;
      if (d > 0 && want <= room) page += ((want + ps - 1) >> a.shift) - have;
      if (d < 0) back += have - ((max(want, static_cast<int64_t>(0)) + ps - 1) >> a.shift);
      page_end[b] = clamp32(page);
      back_end[b] = clamp32(back);
    }
  }
  int64_t tok_all, page_all = 0, back_all = 0;
  const int64_t tok_before = block_scan(tok, red, tok_all) - tok;
  int64_t page_before = 0, back_before = 0;
  if (STEP) {
    page_before = block_scan(page, red, page_all) - page;
    back_before = block_scan(back, red, back_all) - back;
  }
  int taken = 0, errors = 0;
  int64_t page_run = 0;
  tok = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t d = a.delta[b];
    tok += max(d, static_cast<int64_t>(0));
    const int64_t t_end = tok_before + tok;
    tok_end[b] = clamp32(t_end);
    if (STEP) {
      const int64_t len = min(max(static_cast<int64_t>(a.lens[b]), static_cast<int64_t>(0)), room);
      const int64_t want = len + d;
      const int64_t have = (len + ps - 1) >> a.shift;
      const bool fits = d > 0 && want <= room;
      const int64_t need = fits ? ((want + ps - 1) >> a.shift) - have : 0;
      page_run += need;
      const int64_t p_end = page_before + page_run;
      page_end[b] = clamp32(p_end);
      back_end[b] = clamp32(back_before + back_end[b]);
      const bool ok = fits && t_end <= a.tokens && (need == 0 || p_end <= count);
      if (ok) taken += static_cast<int>(need);
      if (d > 0 && !ok)
        errors |= !fits ? DSV2_DEVERR_CACHE_FULL : (t_end > a.tokens ? DSV2_DEVERR_TOKENS : DSV2_DEVERR_NO_PAGE);
      meta[b] = static_cast<uint32_t>(len) | (ok ? 0x80000000u : 0u);
      if (blockIdx.x == 0) a.state_out[b] = static_cast<int>(d < 0 ? max(want, static_cast<int64_t>(0)) : (ok ? want : len));
    } else if (t_end > a.tokens && d > 0) {
      errors |= DSV2_DEVERR_TOKENS;
    }
  }
  if (STEP && taken) atomicAdd(&taken_sum, taken);
  __syncthreads();
  const int used = STEP ? taken_sum : 0;
  // a ring that already holds every page it could get back was not this table's: what does not fit is dropped
  const int given = STEP ? static_cast<int>(min(back_all, static_cast<int64_t>(a.pages - count))) : 0;
  if (blockIdx.x == 0) {
    if (STEP && tid == 0) {
      const int64_t h = static_cast<int64_t>(head) + used;
      a.state_out[a.n] = static_cast<int>(h >= a.pages ? h - a.pages : h);
      a.state_out[a.n + 1] = count - used + given;
      if (given < back_all) errors |= DSV2_DEVERR_BAD_SLOT;
    }
    if (errors && a.status) atomicOr(a.status, errors);
  }

  const int first = blockIdx.x * 256 + tid, stride = gridDim.x * 256;
  const int live = static_cast<int>(min(tok_all, static_cast<int64_t>(a.tokens)));
  int bad = 0;
  for (int i = first; i < a.tokens; i += stride) {
    int slot = -1, pos = -1, row = -1;
    if (i < live) {
      const int b = owner(tok_end, a.n, i);
      const int j = i - (b ? tok_end[b - 1] : 0);
      if (STEP) {
        if (meta[b] & 0x80000000u) {
          const int len = meta[b] & 0x7fffffffu;
          pos = len + j;
          row = b;
          const int have = static_cast<int>((static_cast<int64_t>(len) + ps - 1) >> a.shift);
          const int idx = pos >> a.shift;
          int p;
          if (idx < have) {
            p = a.table[b * a.ts + idx];
          } else {
            int64_t k = static_cast<int64_t>(head) + (b ? page_end[b - 1] : 0) + idx - have;
            p = a.ring[k >= a.pages ? k - a.pages : k];
          }
          if (p >= 0 && p < a.pages)
            slot = (p << a.shift) | (pos & (ps - 1));
          else
            bad = DSV2_DEVERR_BAD_SLOT;
        }
      } else {
        const int64_t t = static_cast<int64_t>(a.lens[b]) + j;
        if (a.lens[b] >= 0 && t < room) {
          pos = static_cast<int>(t);
          row = b;
          const int p = a.table[b * a.ts + (pos >> a.shift)];
          if (p >= 0 && p <= (INT32_MAX >> a.shift))
            slot = (p << a.shift) | (pos & (ps - 1));
          else
            bad = DSV2_DEVERR_BAD_SLOT;
        } else {
          bad = DSV2_DEVERR_BAD_SLOT;
        }
      }
    }
    a.slots[i] = slot;
    a.positions[i] = pos;
    a.rows[i] = row;
  }
  if (bad && a.status) atomicOr(a.status, bad);
  if (!STEP) return;
  for (int k = first; k < used; k += stride) {
    const int b = owner(page_end, a.n, k);
    const int have = static_cast<int>((static_cast<int64_t>(meta[b] & 0x7fffffffu) + ps - 1) >> a.shift);
    const int64_t at = static_cast<int64_t>(head) + k;
    a.table[b * a.ts + have + k - (b ? page_end[b - 1] : 0)] = a.ring[at >= a.pages ? at - a.pages : at];
  }
  for (int k = first; k < given; k += stride) {
    const int b = owner(back_end, a.n, k);
    const int before = b ? back_end[b - 1] : 0;
    const int have = static_cast<int>((static_cast<int64_t>(meta[b] & 0x7fffffffu) + ps - 1) >> a.shift);
    const int kept = have - (back_end[b] - before);
    int64_t at = static_cast<int64_t>(head) + count + k;  // < 3 * pages: head and count are at most pages each
    while (at >= a.pages) at -= a.pages;
    a.ring[at] = a.table[b * a.ts + kept + k - before];
  }
}

static int plan_launch(const char* what, bool step, const PlanArgs& a, int page_size, void* stream) {
  DSV2_REQUIRE(a.n >= 0 && a.n <= kMaxRequests, DSV2_E_SHAPE, "%s: %d requests, at most %d", what, a.n, kMaxRequests);
  DSV2_REQUIRE(a.shift >= 0, DSV2_E_SHAPE, "%s: page_size %d is no power of two in [1, 1024]", what, page_size);
  DSV2_REQUIRE(a.width > 0 && a.width <= (INT32_MAX >> a.shift) && a.ts >= a.width, DSV2_E_SHAPE,
               "%s: block table of %d columns", what, a.width);
  DSV2_REQUIRE(a.tokens >= 0, DSV2_E_SHAPE, "%s: max_tokens %d", what, a.tokens);
  const int items = a.tokens > a.n ? a.tokens : a.n;
  int wgs = (items + 255) / 256;
  wgs = wgs < 1 ? 1 : (wgs > kPlanWgs ? kPlanWgs : wgs);
  const size_t lds = static_cast<size_t>(a.n) * (step ? 16 : 4);
  if (step)
    hipLaunchKernelGGL(paged_plan_kernel<true>, dim3(wgs), dim3(256), lds, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(paged_plan_kernel<false>, dim3(wgs), dim3(256), lds, (hipStream_t)stream, a);
  return dsv2_launch_status(what);
}

extern "C" int dsv2_paged_step(const int32_t* state, const int32_t* delta, int requests, int32_t* block_table,
                               int64_t table_stride, int table_width, int32_t* free_pages, int n_pages, int page_size,
                               int max_tokens, int32_t* state_out, int32_t* slots, int32_t* positions, int32_t* rows,
                               int32_t* status, void* stream) {
  DSV2_REQUIRE(state && delta && block_table && free_pages && state_out && (max_tokens == 0 || (slots && positions && rows)),
               DSV2_E_NULL, "paged_step: null pointer");
  const int shift = page_shift(page_size);
  DSV2_REQUIRE(n_pages > 0 && (shift < 0 || n_pages <= (INT32_MAX >> shift)), DSV2_E_SHAPE, "paged_step: %d pages",
               n_pages);
  DSV2_REQUIRE(state_out + requests + 2 <= state || state + requests + 2 <= state_out, DSV2_E_SHAPE,
               "paged_step: state_out overlaps state");
  const PlanArgs a{state, delta, requests, block_table, table_stride, table_width, free_pages, n_pages,
                   shift, max_tokens, state_out, slots, positions, rows, status};
  return plan_launch("paged_step", true, a, page_size, stream);
}

extern "C" int dsv2_paged_slots(const int32_t* starts, const int32_t* counts, int requests, const int32_t* block_table,
                                int64_t table_stride, int table_width, int page_size, int max_tokens, int32_t* slots,
                                int32_t* positions, int32_t* rows, int32_t* status, void* stream) {
  DSV2_REQUIRE(starts && counts && block_table && (max_tokens == 0 || (slots && positions && rows)), DSV2_E_NULL,
               "paged_slots: null pointer");
  const PlanArgs a{starts, counts, requests, const_cast<int32_t*>(block_table), table_stride, table_width, nullptr, 0,
                   page_shift(page_size), max_tokens, nullptr, slots, positions, rows, status};
  return plan_launch("paged_slots", false, a, page_size, stream);
}

// ---------------------------------------------------------------------------
// Rows into pages and back: one wave a token, a lane 8 latent values (4 lanes a block)
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
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, v.x), scale, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, v.y), scale, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, v.z), scale, 2);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, v.w), scale, 3);
  const TokenAt at = token_at(slot, shift, page_stride);
  *reinterpret_cast<uint32_t*>(pages + at.code + lane * 4) = odd ? 0u : code;
  if (lane < 8) *reinterpret_cast<uint4*>(pages + at.rope + lane * 16) = k;
  if ((lane & 3) == 0) pages[at.scale + (lane >> 2)] = static_cast<uint8_t>(s);
}

__global__ __launch_bounds__(256) void paged_read_kernel(const uint8_t* __restrict__ pages, int64_t page_stride,
                                                         int n_slots, int shift, const int32_t* __restrict__ slots,
                                                         int n, bf16_t* __restrict__ out, int64_t os,
                                                         int32_t* __restrict__ status) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= n) return;
  const int slot = slots[r];
  bf16_t* row = out + r * os;
  uint4 v = make_uint4(0, 0, 0, 0), k = v;
  if (slot >= 0 && slot < n_slots) {
    const TokenAt at = token_at(slot, shift, page_stride);
    const uint32_t code = *reinterpret_cast<const uint32_t*>(pages + at.code + lane * 4);
    const uint32_t s = pages[at.scale + (lane >> 2)];
    if (lane < 8) k = ldg16(pages + at.rope + lane * 16);
    v = decode8(code, s);
    if (s == kNanScale) v = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
  } else if (slot >= n_slots && lane == 0 && status) {
    atomicOr(status, DSV2_DEVERR_BAD_SLOT);
  }
  *reinterpret_cast<uint4*>(row + lane * 8) = v;
  if (lane < 8) *reinterpret_cast<uint4*>(row + kLat + lane * 8) = k;
}

extern "C" int dsv2_paged_write_fp4(const void* rows, int64_t row_stride, int n, const int32_t* slots, void* pages,
                                    int64_t page_stride, int n_pages, int page_size, int32_t* status, void* stream) {
  if (const int rc = paged_check_pool("paged_write_fp4", pages, page_stride, n_pages, page_size)) return rc;
  DSV2_REQUIRE(n >= 0 && row_stride >= kRow, DSV2_E_SHAPE, "paged_write_fp4: bad shape");
  if (n == 0) return DSV2_OK;
  DSV2_REQUIRE(rows && slots, DSV2_E_NULL, "paged_write_fp4: null pointer");
  DSV2_REQUIRE(dsv2_aligned16(rows) && row_stride % 8 == 0, DSV2_E_ALIGN, "paged_write_fp4: rows alignment");
  const int shift = page_shift(page_size);
  hipLaunchKernelGGL(paged_write_kernel, dim3((n - 1) / 4 + 1), dim3(256), 0, (hipStream_t)stream, (const bf16_t*)rows,
                     row_stride, n, slots, (uint8_t*)pages, page_stride, n_pages << shift, shift, status);
  return dsv2_launch_status("paged_write_fp4");
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
  hipLaunchKernelGGL(paged_read_kernel, dim3((n - 1) / 4 + 1), dim3(256), 0, (hipStream_t)stream,
                     (const uint8_t*)pages, page_stride, n_pages << shift, shift, slots, n, (bf16_t*)out, out_stride,
                     status);
  return dsv2_launch_status("paged_read_fp4");
}
