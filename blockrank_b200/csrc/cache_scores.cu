// Document scores from the 4-bit cache: the signal rows against the held keys of every document.
//
// A CTA takes some of a prompt's documents, about as many pages as every other CTA, for one KV head and up to 8 kTiles (head, signal
// row) pairs; its warps take equal parts of those pages, whatever documents they belong to, and keep a running (maximum, sum) per
// pair and document.  The pairs of a prompt's documents are merged by the kernel that merges those of doc_scores.
// The floor is the read of the keys (72 bytes per token and KV head at head_dim 128); bound by instructions, as the attention of few rows
// is.  16 prompts of 100 documents of 32 to 256 tokens, two rows of 32 heads on 8: 49 us, 2.6 TB/s; one prompt of 5 documents
// 8.6.  (Up to 64 documents at a time, not 32, so that no CTA has a second batch: 48.5 and 9.2; two batches as long as each other:
// 49.6.)
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "cache_layout.cuh"
#include "score_args.cuh"
#include "tc_ptx.cuh"

namespace brk {
namespace {

using namespace cache;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 3;  // pages (their K parts) a warp has in shared memory
constexpr int kDocs = 32;   // documents at a time: one per lane
constexpr float kLog2e = 1.4426950408889634f;

struct CacheScoreArgs {
  const unsigned char* pages;
  View q;  // (B, N, R, D)
  const int32_t* table;
  const int32_t* blk_start;
  const int32_t* blk_len;
  float2* partial;  // [B, N, R, M - 2]
  int32_t* status;
  int n_pages, N, Nk, R, M, P, max_block_len;
  float scale;
};

__device__ __forceinline__ float2 merged(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x), ref = top == -INFINITY ? 0.f : top;
  return make_float2(top, a.y * ptx::ex2(a.x - ref) + b.y * ptx::ex2(b.x - ref));
}

template <typename T, int D, int kTiles>
__global__ void __launch_bounds__(kThreads, kTiles == 1 && sizeof(T) == 2 ? 3 : 2) cache_scores_kernel(CacheScoreArgs a) {
  using L = Layout<D>;
  constexpr int kCols = 8 * kTiles;
  extern __shared__ __align__(16) unsigned char smem[];  // [kWarps][kStages][K part of a page]
  __shared__ float2 s_ml[kWarps][kDocs][kCols];
  __shared__ int s_scan[kWarps], s_before[2];
  __shared__ int2 s_span[kThreads];      // (start, length) of the first documents
  __shared__ int32_t s_table[kThreads];  // the first page numbers
  ptx::grid_dependency_wait();
  ptx::grid_dependency_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.y / a.Nk, kvh = blockIdx.y % a.Nk, row0 = blockIdx.z * kCols;
  const int G = a.N / a.Nk, GR = G * a.R, nd = a.M - 2;
  const int32_t *const bs = a.blk_start + (int64_t)b * a.M, *const bl = a.blk_len + (int64_t)b * a.M;

  const int32_t* const table = a.table + (int64_t)b * a.P;

  // document d's span (length 0 if it is malformed) and its pages
  auto span = [&](int d, int& start, int& len) {
    start = bs[d + 1];
    len = bl[d + 1];
    if (span_is_bad(bs, bl, d + 1, (int64_t)a.P * kPage) || len > a.max_block_len) {
      if (a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);
      len = 0;
    }
  };
  auto pages_of = [](int start, int len) { return len > 0 ? (start + len - 1) / kPage - start / kPage + 1 : 0; };
  auto warp_scan = [&](int x) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    return x;
  };

  // ---- this CTA's documents: those whose first page is in its share of all documents' pages ----
  int my_start = 0, my_len = 0;
  s_table[tid] = tid < a.P ? table[tid] : -1;
  if (tid < nd) span(tid, my_start, my_len);
  s_span[tid] = make_int2(my_start, my_len);
  typename QueryRows<T, D, kTiles>::Raw raw;
  QueryRows<T, D, kTiles>::fetch([&](int c) -> const T* {
    const int r = row0 + c;
    if (r >= GR) return nullptr;
    return reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb + (int64_t)(kvh * G + r / a.R) * a.q.sh + (int64_t)(r % a.R) * a.q.ss;
  }, g, t, raw);
  int64_t lo = 0, hi = 0;
  if (tid < 2) s_before[tid] = 0;
  // All pages (pass 0); then the number of documents that begin before the share, and before its end.  Up to kThreads documents are
  // looked at once.
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int64_t before = 0;
#pragma unroll 1
    for (int d0 = 0; d0 < nd; d0 += kThreads) {
      int st = my_start, ln = my_len;
      if (d0 > 0 && d0 + tid < nd) span(d0 + tid, st, ln);
      const int n = d0 + tid < nd ? pages_of(st, ln) : 0, x = warp_scan(n);
      if (lane == 31) s_scan[warp] = x;
      __syncthreads();
      int sum = 0, first = x - n;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) first += s_scan[w];
        sum += s_scan[w];
      }
      const bool only = nd <= kThreads;
      if (only) {
        lo = (int64_t)sum * blockIdx.x / gridDim.x;
        hi = (int64_t)sum * (blockIdx.x + 1) / gridDim.x;
      }
      if (pass == 1 || only) {
        const unsigned below = __ballot_sync(0xffffffffu, d0 + tid < nd && before + first < lo);
        const unsigned below_end = __ballot_sync(0xffffffffu, d0 + tid < nd && (before + first < hi || blockIdx.x + 1 == gridDim.x));
        if (lane == 0) {
          atomicAdd(&s_before[0], __popc(below));
          atomicAdd(&s_before[1], __popc(below_end));
        }
        if (only) pass = 1;
      }
      before += sum;
      __syncthreads();
    }
    if (pass == 0) {
      lo = before * blockIdx.x / gridDim.x;
      hi = before * (blockIdx.x + 1) / gridDim.x;
    }
  }
  const int doc_end = s_before[1];

  QueryRows<T, D, kTiles> q;
  q.make(raw, g, t);
  float sl2[kTiles][2], mx[kTiles][2], sum[kTiles][2];  // this lane's keys
#pragma unroll
  for (int c = 0; c < kTiles; ++c)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      sl2[c][x] = a.scale * kLog2e * q.unit[c][x];
      mx[c][x] = -INFINITY;
      sum[c][x] = 0.f;
    }
  unsigned char* const ring = smem + warp * kStages * L::kHalf;
  const unsigned char* const head = a.pages + (int64_t)kvh * L::kBytes;
  auto page_number = [&](int i) { return i < kThreads ? s_table[i] : table[i]; };

#pragma unroll 1
  for (int doc0 = s_before[0]; doc0 < doc_end; doc0 += kDocs) {
    const int n_docs = min(kDocs, doc_end - doc0);
    int start = 0, len = 0;  // lane l: of document doc0 + l
    if (lane < n_docs) {
      if (doc0 + lane < kThreads) {
        start = s_span[doc0 + lane].x;
        len = s_span[doc0 + lane].y;
      } else {
        span(doc0 + lane, start, len);
      }
    }
    const int n = pages_of(start, len);
    const int end = warp_scan(n), pages = __shfl_sync(0xffffffffu, end, 31);
    const int from = (int)((int64_t)pages * warp / kWarps), to = (int)((int64_t)pages * (warp + 1) / kWarps);
    for (int i = lane; i < kDocs * kCols; i += 32) (&s_ml[warp][0][0])[i] = make_float2(-INFINITY, 0.f);
    __syncwarp();

    // A walk over the pages from .. to - 1; page numbers are read one page before they are needed, pages kStages - 1 before.
    struct Walk {
      int at, doc, next, slot0, start, len;  // page at is of document doc0 + doc, as are all before next; its first slot
    };
    auto enter = [&](Walk& w) {  // the document of page w.at
      w.doc = __popc(__ballot_sync(0xffffffffu, end <= w.at));
      w.next = __shfl_sync(0xffffffffu, end, w.doc);
      w.start = __shfl_sync(0xffffffffu, start, w.doc);
      w.len = __shfl_sync(0xffffffffu, len, w.doc);
      w.slot0 = (w.start / kPage + w.at - (w.next - __shfl_sync(0xffffffffu, n, w.doc))) * kPage;
    };
    auto step = [&](Walk& w) {
      ++w.at;
      w.slot0 += kPage;
      if (w.at < to && w.at >= w.next) enter(w);
    };
    Walk ahead = {from, 0, 0, 0, 0, 0}, here = ahead;
    if (from < to) {
      enter(ahead);
      here = ahead;
    }
    int id = from < to ? page_number(ahead.slot0 / kPage) : 0;
    uint32_t absent = 0;  // bit s: the page in stage s does not exist
    auto request = [&](int stage) {
      if (ahead.at < to) {
        const int page = id;
        step(ahead);
        if (ahead.at < to) id = page_number(ahead.slot0 / kPage);
        if (page >= 0 && page < a.n_pages) {
          absent &= ~(1u << stage);
          const unsigned char* src = head + (int64_t)page * a.Nk * L::kBytes;
          for (int x = lane * 16; x < L::kHalf; x += 512) cp_async16(ring + stage * L::kHalf + x, src + x);
        } else {
          absent |= 1u << stage;
          if (lane == 0 && a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) request(s);

    int stage = 0;
#pragma unroll 1
    while (here.at < to) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      request(stage == 0 ? kStages - 1 : stage - 1);  // into the place of the page before
      if (!((absent >> stage) & 1)) {
        float s[kTiles][4][4];
        const int first = here.start - here.slot0, last = first + here.len;  // the document's tokens in this page
        q.logits(ring + stage * L::kHalf, g, t, s);
        if (first > 0 || last < kPage) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int key = 16 * k + 8 * y + g;
              if (key < first || key >= last) {
#pragma unroll
                for (int c = 0; c < kTiles; ++c) s[c][k][2 * y] = s[c][k][2 * y + 1] = -INFINITY;
              }
            }
        }
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float top = mx[c][x];
#pragma unroll
            for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(s[c][k][x], s[c][k][2 + x]));
            const float ref = top == -INFINITY ? 0.f : top * sl2[c][x];
            sum[c][x] *= ptx::ex2(mx[c][x] * sl2[c][x] - ref);
            mx[c][x] = top;
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int y = 0; y < 2; ++y) sum[c][x] += ptx::ex2(fmaf(s[c][k][2 * y + x], sl2[c][x], -ref));
          }
      }
      stage = stage + 1 == kStages ? 0 : stage + 1;
      const int doc = here.doc;
      step(here);
      if (here.at >= to || here.doc != doc) {  // the last of this warp's pages of the document
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float2 ml = make_float2(mx[c][x] * sl2[c][x], sum[c][x]);
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1)
              ml = merged(ml, make_float2(__shfl_xor_sync(0xffffffffu, ml.x, off), __shfl_xor_sync(0xffffffffu, ml.y, off)));
            if (g == 0) s_ml[warp][doc][8 * c + 2 * t + x] = ml;
            mx[c][x] = -INFINITY;
            sum[c][x] = 0.f;
          }
      }
    }
    cp_async_wait<0>();
    __syncthreads();
    for (int i = tid; i < kDocs * kCols; i += kThreads) {
      const int doc = i % kDocs, r = row0 + i / kDocs;
      if (doc >= n_docs || r >= GR) continue;
      float2 ml = s_ml[0][doc][i / kDocs];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) ml = merged(ml, s_ml[w][doc][i / kDocs]);
      a.partial[(((int64_t)b * a.N + kvh * G + r / a.R) * a.R + r % a.R) * nd + doc0 + doc] = ml;
    }
    __syncthreads();
  }
}

}  // namespace

size_t cache_scores_workspace(const brk_cache_score_params& p) { return (size_t)p.B * p.N * p.R * (p.M - 2) * sizeof(float2); }

int cache_scores_launch(const brk_cache_score_params& p, void* ws, cudaStream_t st) {
  CacheScoreArgs a;
  a.pages = static_cast<const unsigned char*>(p.cache.pages);
  a.q = make_view(p.q);
  a.table = p.page_table;
  a.blk_start = p.blk_start;
  a.blk_len = p.blk_len;
  a.partial = static_cast<float2*>(ws);
  a.status = p.status;
  a.n_pages = p.cache.n_pages; a.N = p.N; a.Nk = p.cache.Nk; a.R = p.R; a.M = p.M; a.P = p.P;
  a.max_block_len = p.max_block_len;
  a.scale = p.scale;
  const int nd = p.M - 2, rows = p.N / a.Nk * p.R, tiles = rows > 8 ? 2 : 1;
  const int z = (rows + 8 * tiles - 1) / (8 * tiles);
  // Shares of a prompt's documents, at least a page for each warp: a round of CTAs takes as long as its share, with about eight pages' time
  // for beginning and end.
  const int64_t ctas = (int64_t)p.B * a.Nk * z, room = (tiles == 1 && p.dtype == BRK_BF16 ? 3 : 2) * (int64_t)std::max(1, sm_count());
  const int64_t most = std::min<int64_t>(nd, (p.P + kWarps - 1) / kWarps);
  int64_t shares = 1, best = INT64_MAX;
  for (int64_t round = 0; round <= 8; ++round) {  // (the most shares of so many rounds, and the fewest)
    const int64_t s = std::min(most, std::max<int64_t>(1, round * room / ctas));
    const int64_t cost = (ctas * s + room - 1) / room * ((p.P + s - 1) / s + 8);
    if (cost < best) {
      best = cost;
      shares = s;
    }
  }
  const dim3 grid((unsigned)shares, p.B * a.Nk, z);
  auto run = [&](auto kern, std::atomic<bool>* configured) -> int {
    const int bytes = kWarps * kStages * (int)head_page_bytes(p.cache.D) / 2;
    int dev = 0;
    BRK_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
      BRK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      BRK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared));
      if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    return launch_dependent(kern, grid, dim3(kThreads), bytes, st, a);
  };
  static std::atomic<bool> done[8][64] = {};
  auto of_head_dim = [&](auto d, std::atomic<bool>(*flags)[64]) -> int {
    constexpr int D = decltype(d)::value;
    if (p.dtype == BRK_F32) return tiles == 1 ? run(cache_scores_kernel<float, D, 1>, flags[0]) : run(cache_scores_kernel<float, D, 2>, flags[1]);
    return tiles == 1 ? run(cache_scores_kernel<__nv_bfloat16, D, 1>, flags[2]) : run(cache_scores_kernel<__nv_bfloat16, D, 2>, flags[3]);
  };
  const int rc = p.cache.D == 128 ? of_head_dim(std::integral_constant<int, 128>(), done) : of_head_dim(std::integral_constant<int, 64>(), done + 4);
  if (rc) return rc;
  ScoreArgs m = {};
  m.partial = a.partial;
  m.mass = p.doc_mass;
  m.logits = p.logits;
  m.inv_count_temp = 1.f / ((float)(p.N * p.R) * p.temperature);
  m.B = p.B; m.N = p.N; m.Nk = a.Nk; m.M = p.M; m.R = p.R;
  return doc_merge_launch(m, st);
}

}  // namespace brk
