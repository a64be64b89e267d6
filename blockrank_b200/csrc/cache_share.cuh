// What the kernels of the cache's attention share: their arguments, and a CTA's share of a prompt's pages.
#pragma once
#include "cache_layout.cuh"
#include "tc_ptx.cuh"

namespace brk {
namespace cache {

constexpr int kManyShare = 256;  // pages a CTA of the tcgen05 kernel takes at most
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct CacheAttnArgs {
  const unsigned char* pages;
  View q, o;  // (B, N, Lq, D)
  const int32_t* table;  // [B, P]
  const int32_t* blk_start;
  const int32_t* blk_len;
  const int32_t* q_len;  // [B] or null: Lq each
  float* lse;            // [B, N, Lq] or null
  int32_t* status;
  float* part_o;         // [B, N, Lq, shares, D]
  float2* part_ml;       // [B, N, Lq, shares] (maximum in log2 units, sum)
  int n_pages, B, N, Nk, Lq, M, P, shares;
  bool cluster;          // a prompt's shares are a cluster, which joins its parts itself
  float scale;
  Codes codes;
};

struct Share {
  int rows;        // of the prompt
  int n_rows;      // of this CTA; none is left where it is not positive
  int first_slot;  // slot of the prompt's row 0
  int page0, n;    // the CTA's pages: entries page0 .. page0 + n - 1 of the page table
  bool bad;        // spans or number of rows malformed: the prompt has no rows
};

// Rows row0 .. row0 + max_rows - 1 of prompt b (query heads of a group at one token after the other) against an even share, of at
// least min_pages, of the pages up to the last row's slot.  s_mask [2 kShare]: which tokens of these pages lie in a block; s_page [kShare]: the pages'
// numbers, -1 for one without such a token.  The latencies are paid once each: spans and number of rows, with what `meanwhile` requests and
// the first entries of the page table; the other entries.
template <int kThreads, int kShare, typename F>
__device__ __forceinline__ Share find_share(const CacheAttnArgs& a, int b, int row0, int max_rows, int share, int min_pages, uint32_t* s_mask,
                                            int32_t* s_page, F meanwhile) {
  const int tid = threadIdx.x, G = a.N / a.Nk;
  const int32_t *start = a.blk_start + (int64_t)b * a.M, *len = a.blk_len + (int64_t)b * a.M, *table = a.table + (int64_t)b * a.P;
  const int64_t slots = (int64_t)a.P * kPage;
  const int last_start = start[a.M - 1], last_len = len[a.M - 1], given = a.q_len ? a.q_len[b] : a.Lq;
  __shared__ int32_t s_table[kThreads];
  __shared__ int2 s_span[kThreads];  // (start, length) of the first blocks
  s_table[tid] = tid < a.P ? table[tid] : -1;
  meanwhile();
  bool bad = given < 0 || given > a.Lq || given > last_len;
  for (int m = tid; m < a.M; m += kThreads) {
    bad |= span_is_bad(start, len, m, slots);
    if (m < kThreads) s_span[m] = make_int2(start[m], len[m]);
  }
  Share r;
  r.bad = __syncthreads_or(bad);
  if (r.bad && tid == 0 && a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);

  auto block = [&](int m) { return m < kThreads ? s_span[m] : make_int2(start[m], len[m]); };
  r.rows = r.bad ? 0 : given;
  r.n_rows = min(r.rows * G - row0, max_rows);
  r.first_slot = r.bad ? 0 : last_start + last_len - r.rows;
  const int live = r.n_rows > 0 ? (r.first_slot + (row0 + r.n_rows - 1) / G) / kPage + 1 : 0;
  const int per = max((live + a.shares - 1) / a.shares, min(live, min_pages));
  r.page0 = min(live, share * per);
  r.n = min(live, r.page0 + per) - r.page0;
  for (int i = tid; i < r.n; i += kThreads) {
    const int at = r.page0 + i, lo = at * kPage;
    int page = at < kThreads ? s_table[at] : table[at];
    int m = 0;  // the first block that ends behind the page's first token (blocks are in order)
    for (int size = a.M; size > 0;) {
      const int half = size / 2;
      const int2 x = block(m + half);
      if (x.x + x.y <= lo) {
        m += half + 1;
        size -= half + 1;
      } else {
        size = half;
      }
    }
    uint32_t w[2] = {0, 0};
    for (; m < a.M; ++m) {
      const int2 x = block(m);
      if (x.x >= lo + kPage) break;
      const int from = max(x.x - lo, 0), to = min(x.x + x.y - lo, kPage);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int f = max(from - 32 * h, 0), t = min(to - 32 * h, 32);
        if (f < t) w[h] |= (t == 32 ? ~0u : (1u << t) - 1) & (~0u << f);
      }
    }
    const bool needed = (w[0] | w[1]) != 0;
    if (needed && (page < 0 || page >= a.n_pages)) {
      if (a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);
      page = -1;
    }
    s_mask[2 * i] = w[0];
    s_mask[2 * i + 1] = w[1];
    s_page[i] = needed ? page : -1;
  }
  __syncthreads();
  return r;
}

}  // namespace cache

int cache_attn_tc_launch(const cache::CacheAttnArgs& a, int D, cudaStream_t st);

}  // namespace brk
