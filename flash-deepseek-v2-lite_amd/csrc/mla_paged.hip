// Absorbed-MLA attention over the paged latent cache held in 4 bits.
//
//   s_t = scale * q . (latent_t | rope_t),  p = softmax(s),  o = sum_t p_t latent_t
//
// One (query token, head) pair is a column; a request's columns are numbered token by token, and 16 of
// them make the narrow side of v_mfma_f32_16x16x32_bf16 (S^T = K Q^T, O^T += V^T P^T).
#include "paged.h"

using namespace paged;

namespace {
constexpr int kTile = 32;
constexpr int kLdsRow = kRow + 8;

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
  float scale_log2;
  bf16_t* out;
  int64_t o_ts, o_hs;
  int32_t* status;
};
}  // namespace

__global__ __launch_bounds__(256) void mla_paged_kernel(const PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) bf16_t lds[kTile * kLdsRow];
  __shared__ floatx4_t spart[4][64];
  const int b = blockIdx.y, c0 = blockIdx.x * 16;
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, li = lane & 15, kg = lane >> 4;
  const int q0 = a.cu_q ? a.cu_q[b] : b;
  const int q1 = a.cu_q ? a.cu_q[b + 1] : b + 1;
  const int nq = q0 >= 0 ? max(min(q1, a.tokens) - q0, 0) : 0;
  const int columns = min(nq, a.max_q) * a.heads;
  if (nq > a.max_q && blockIdx.x == 0 && threadIdx.x == 0 && a.status) atomicOr(a.status, DSV2_DEVERR_TOKENS);
  if (c0 >= columns) return;
  const int room = static_cast<int>(min(static_cast<int64_t>(a.width) << a.shift, static_cast<int64_t>(INT32_MAX)));
  const int len = min(max(a.lens[b], 0), room);
  const int col = c0 + li;
  const bool live = col < columns;
  const int j = live ? col / a.heads : 0, h = live ? col - j * a.heads : 0;
  const int seen = live ? max(len - nq + j + 1, 0) : 0;
  const int jl = min(c0 + 15, columns - 1) / a.heads;
  const int most = max(len - nq + jl + 1, 0);
  const bf16_t* qc = a.q + (q0 + j) * a.q_ts + h * a.q_hs;
  const int sblk = wv >> 1, k0 = (wv & 1) * 9;
  bf16x8_t qf[9];
#pragma unroll
  for (int kk = 0; kk < 9; ++kk) qf[kk] = as_bf16x8(keep_if(live, ldg16(qc + kg * 8 + (k0 + kk) * 32)));

  float m_run = -__FLT_MAX__, l_run = 0.f;
  floatx4_t acc[8];
#pragma unroll
  for (int mb = 0; mb < 8; ++mb) acc[mb] = floatx4_t{0.f, 0.f, 0.f, 0.f};
  for (int t0 = 0; t0 < most; t0 += kTile) {
    __syncthreads();
    const int tok = tid >> 3, part = tid & 7, t = t0 + tok;
    int page = -1;
    if (t < most) {
      page = a.table[b * a.ts + (t >> a.shift)];
      if (page < 0 || page >= a.n_pages) {
        if (part == 0 && a.status) atomicOr(a.status, DSV2_DEVERR_BAD_SLOT);
        page = -1;
      }
    }
    uint4 k = make_uint4(0, 0, 0, 0), code[2] = {k, k};
    uint32_t s[2] = {127, 127};
    if (page >= 0) {
      const TokenAt at = token_at((page << a.shift) | (t & ((1 << a.shift) - 1)), a.shift, a.page_stride);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        code[i] = ldg16(a.pages + at.code + (part * 2 + i) * 16);
        s[i] = a.pages[at.scale + part * 2 + i];
      }
      k = ldg16(a.pages + at.rope + part * 16);
      // a block of NaN: its codes are 0, and one rotary key becomes NaN instead, so that only the
      // queries that see the token get NaN (a latent NaN times an unseen token's p = 0 would be one too)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (s[i] == kNanScale) {
          s[i] = 127;
          k.x = 0x7fc07fc0u;
        }
    }
    bf16_t* L = lds + tok * kLdsRow;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        *reinterpret_cast<uint4*>(L + (part * 2 + i) * 32 + x * 8) = decode8(w[x], s[i]);
      }
    }
    *reinterpret_cast<uint4*>(L + kLat + part * 8) = k;
    __syncthreads();
    {
      floatx4_t sp = floatx4_t{0.f, 0.f, 0.f, 0.f};
      const bf16_t* kr = lds + (sblk * 16 + li) * kLdsRow + kg * 8 + k0 * 32;
#pragma unroll
      for (int kk = 0; kk < 9; ++kk) sp = mfma16x16x32(*reinterpret_cast<const bf16x8_t*>(kr + kk * 32), qf[kk], sp);
      spart[wv][lane] = sp;
    }
    __syncthreads();
    float p[8], mx = -__FLT_MAX__;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int blk = i >> 2, e = i & 3;
      const float v = (spart[2 * blk][lane][e] + spart[2 * blk + 1][lane][e]) * a.scale_log2;
      p[i] = t0 + blk * 16 + 4 * kg + e < seen ? v : -INFINITY;
      mx = fmaxf(mx, p[i]);
    }
    mx = xor32_max(xor16_max(mx));
    const float m_new = fmaxf(m_run, mx);
    const float alpha = exp2f(m_run - m_new);
    m_run = m_new;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = exp2f(p[i] - m_run);
      sum += p[i];
    }
    l_run = l_run * alpha + xor32_sum(xor16_sum(sum));
    const bf16x8_t pb = as_bf16x8(pack8(p));
    const bf16_t* vp = lds + (4 * kg + (li >> 2)) * kLdsRow + wv * 128 + 4 * (li & 3);
#pragma unroll
    for (int mb = 0; mb < 8; ++mb) {
      acc[mb] *= alpha;
      const uint2 lo = lds_read_tr16(vp + mb * 16), hi = lds_read_tr16(vp + mb * 16 + 16 * kLdsRow);
      acc[mb] = mfma16x16x32(as_bf16x8(make_uint4(lo.x, lo.y, hi.x, hi.y)), pb, acc[mb]);
    }
  }
  if (!live) return;
  const float inv = seen > 0 ? 1.0f / l_run : 0.f;
  bf16_t* o = a.out + (q0 + j) * a.o_ts + h * a.o_hs + wv * 128 + 4 * kg;
#pragma unroll
  for (int mb = 0; mb < 8; ++mb)
    *reinterpret_cast<uint2*>(o + mb * 16) =
        make_uint2(pack2(acc[mb][0] * inv, acc[mb][1] * inv), pack2(acc[mb][2] * inv, acc[mb][3] * inv));
}

extern "C" int64_t dsv2_mla_paged_workspace_size(int requests, int max_q, int heads, int table_width, int page_size) {
  return 16;
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
  DSV2_REQUIRE(dsv2_aligned16(q) && dsv2_aligned16(out) && q_ts % 8 == 0 && q_hs % 8 == 0 && out_ts % 8 == 0 &&
                   out_hs % 8 == 0,
               DSV2_E_ALIGN, "mla_decode_paged_fp4: alignment");
  if (tokens == 0 || requests == 0) return DSV2_OK;
  DSV2_REQUIRE(workspace && dsv2_aligned16(workspace) &&
                   workspace_bytes >= dsv2_mla_paged_workspace_size(requests, max_q, heads, table_width, page_size),
               DSV2_E_SHAPE, "mla_decode_paged_fp4: workspace of %lld bytes", (long long)workspace_bytes);
  const PagedAttnArgs a{(const bf16_t*)q, q_ts, q_hs, tokens, heads, (const uint8_t*)pages, page_stride, n_pages,
                        page_shift(page_size), block_table, table_stride, table_width, lens, cu_q, cu_q ? max_q : 1,
                        softmax_scale * 1.4426950408889634f, (bf16_t*)out, out_ts, out_hs, status};
  const int tiles = (a.max_q * heads + 15) / 16;
  hipLaunchKernelGGL(mla_paged_kernel, dim3(tiles, requests), dim3(256), 0, (hipStream_t)stream, a);
  return dsv2_launch_status("mla_decode_paged_fp4");
}
