// What the kernels of the cache's attention share: their arguments, and a CTA's share of a prompt's pages.
// A share can be as long as a page table: what a CTA needs to know of its pages it finds out for so many at a time as it has room for.
#pragma once
#include "cache_layout.cuh"
#include "tc_ptx.cuh"

namespace brk {
namespace cache {

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

// Shared memory: the first entries of the prompt's page table and of its block spans (start, length).
template <int kThreads>
struct Prompt {
  int32_t table[kThreads];
  int2 span[kThreads];
};

struct Share {
  int rows;        // of the prompt
  int n_rows;      // of this CTA; none is left where it is not positive
  int first_slot;  // slot of the prompt's row 0
  int page0, n;    // the CTA's pages: entries page0 .. page0 + n - 1 of the page table
  bool bad;        // spans or number of rows malformed: the prompt has no rows
};

struct Lists {  // of a prompt
  const int32_t *start, *len, *table;
};
__device__ __forceinline__ Lists lists_of(const CacheAttnArgs& a, int b) {
  return {a.blk_start + (int64_t)b * a.M, a.blk_len + (int64_t)b * a.M, a.table + (int64_t)b * a.P};
}

// What n entries of the page table from number `from` on say, by `threads` threads of which this is number `me`.  s_mask [2 n]: which tokens
// of the page lie in a block; s_page [n]: its number, -1 for one without such a token.
template <int kThreads>
__device__ __forceinline__ void find_pages(const CacheAttnArgs& a, const Lists& lists, const Prompt<kThreads>& prompt, int from, int n, int me,
                                           int threads, uint32_t* s_mask, int32_t* s_page) {
  auto block = [&](int m) { return m < kThreads ? prompt.span[m] : make_int2(lists.start[m], lists.len[m]); };
  for (int i = me; i < n; i += threads) {
    const int at = from + i, lo = at * kPage;
    int page = at < kThreads ? prompt.table[at] : lists.table[at];
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
}

// Rows row0 .. row0 + max_rows - 1 of prompt b (query heads of a group at one token after the other) against an even share, of at
// least min_pages, of the pages up to the last row's slot; of the first kAtOnce of them what find_pages says.  The latencies are paid once
// each: spans and number of rows, with what `meanwhile` requests and the first entries of the page table; the other entries.
template <int kAtOnce, int kThreads, typename F>
__device__ __forceinline__ Share find_share(const CacheAttnArgs& a, int b, int row0, int max_rows, int share, int min_pages,
                                            Prompt<kThreads>& prompt, uint32_t* s_mask, int32_t* s_page, F meanwhile) {
  const int tid = threadIdx.x, G = a.N / a.Nk;
  const Lists lists = lists_of(a, b);
  const int32_t *start = lists.start, *len = lists.len;
  const int64_t slots = (int64_t)a.P * kPage;
  const int last_start = start[a.M - 1], last_len = len[a.M - 1], given = a.q_len ? a.q_len[b] : a.Lq;
  prompt.table[tid] = tid < a.P ? lists.table[tid] : -1;
  meanwhile();
  bool bad = given < 0 || given > a.Lq || given > last_len;
  for (int m = tid; m < a.M; m += kThreads) {
    bad |= span_is_bad(start, len, m, slots);
    if (m < kThreads) prompt.span[m] = make_int2(start[m], len[m]);
  }
  Share r;
  r.bad = __syncthreads_or(bad);
  if (r.bad && tid == 0 && a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);

  r.rows = r.bad ? 0 : given;
  r.n_rows = min(r.rows * G - row0, max_rows);
  r.first_slot = r.bad ? 0 : last_start + last_len - r.rows;
  const int live = r.n_rows > 0 ? (r.first_slot + (row0 + r.n_rows - 1) / G) / kPage + 1 : 0;
  const int per = max((live + a.shares - 1) / a.shares, min(live, min_pages));
  r.page0 = (int)min((int64_t)live, (int64_t)share * per);
  r.n = min(live, r.page0 + per) - r.page0;
  find_pages(a, lists, prompt, r.page0, min(r.n, kAtOnce), tid, kThreads, s_mask, s_page);
  __syncthreads();
  return r;
}

}  // namespace cache

int cache_attn_tc_launch(const cache::CacheAttnArgs& a, int D, cudaStream_t st);

}  // namespace brk
