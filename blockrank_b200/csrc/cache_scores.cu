// Document scores from the 4-bit cache: the signal rows against the held keys of every document.
//
// A CTA takes some of a prompt's documents, about as many pages as every other CTA, for one KV head and up to 8 kTiles (head, signal
// row) pairs; its warps take equal parts of those pages, whatever documents they belong to, and keep a running (maximum, sum) per
// pair and document.  The pairs of a prompt's documents are merged by the kernel that merges those of doc_scores, or, where a prompt
// has few pages, at the end by the CTAs themselves: one per KV head with all documents, a cluster for a prompt.
// The floor is the read of the keys (72 bytes per token and KV head at head_dim 128).  Bound by latency, as the attention of few rows is: 50 %
// of the issue slots, 45 % of the ALU pipe, where the instructions of products and softmax alone (cache_attn.cu) would take 22 us.
// 16 prompts of 100 documents of 32 to 256 tokens, two rows of 32 heads on 8: 50 us, 2.6 TB/s; one prompt of 5 documents 7.9.  (Up to 64
// documents at a time, not 32, so that no CTA has a second batch: 48.5 and 9.2, where these took 49 and 7.6; two batches as long as each
// other: 49.6.)
// A document is never divided between CTAs: few long ones take as long as the longest does on a CTA per KV head (one prompt of a document
// of 100,000 tokens 317 us, its bytes 9; of four of 8,000 34 us, its bytes 3).
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
constexpr int kHeads = 8;   // KV heads of a prompt that a cluster has, at most
constexpr float kLog2e = 1.4426950408889634f;

struct CacheScoreArgs {
  const unsigned char* pages;
  View q;  // (B, N, R, D)
  const int32_t* table;
  const int32_t* blk_start;
  const int32_t* blk_len;
  float2* partial;  // [B, N, R, M - 2], unless
  bool whole;       // a CTA has all documents of a prompt, and a cluster all KV heads: masses and logits are made here
  float* mass;      // [B, N, R, M - 2]
  float* logits;    // [B, M - 2] or null
  float inv_count_temp;
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
  __shared__ float s_mass[kWarps][kDocs], s_total[kDocs];
  __shared__ int2 s_span[kThreads];      // (start, length) of the first documents
  __shared__ int32_t s_table[kThreads];  // the first page numbers
  ptx::grid_dependency_wait();
  ptx::grid_dependency_launch();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int b = a.whole ? blockIdx.y : blockIdx.y / a.Nk, kvh = a.whole ? blockIdx.x : blockIdx.y % a.Nk, row0 = blockIdx.z * kCols;
  const int share = a.whole ? 0 : blockIdx.x, shares = a.whole ? 1 : gridDim.x;
  const int G = a.N / a.Nk, GR = G * a.R, nd = a.M - 2;
  const int32_t *const bs = a.blk_start + (int64_t)b * a.M, *const bl = a.blk_len + (int64_t)b * a.M;

  const int32_t* const table = a.table + (int64_t)b * a.P;

  // document d's span (length 0 in a prompt with a malformed block, which has no documents) and its pages
  bool bad = false;
  auto span = [&](int d, int& start, int& len) {
    const int2 x = d < kThreads ? s_span[d] : make_int2(bs[d + 1], bl[d + 1]);
    start = x.x;
    len = bad ? 0 : x.y;
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
  s_table[tid] = tid < a.P ? table[tid] : -1;
  for (int m = tid; m < a.M; m += kThreads) {
    const bool doc = m > 0 && m < a.M - 1;
    bad |= span_is_bad(bs, bl, m, (int64_t)a.P * kPage) || (doc && bl[m] > a.max_block_len);
    if (doc && m <= kThreads) s_span[m - 1] = make_int2(bs[m], bl[m]);
  }
  typename QueryRows<T, D, kTiles>::Raw raw;
  QueryRows<T, D, kTiles>::fetch([&](int c) -> const T* {
    const int r = row0 + c;
    if (r >= GR) return nullptr;
    return reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb + (int64_t)(kvh * G + r / a.R) * a.q.sh + (int64_t)(r % a.R) * a.q.ss;
  }, g, t, raw);
  int64_t lo = 0, hi = 0;
  if (tid < 2) s_before[tid] = 0;
  bad = __syncthreads_or(bad);
  if (bad && tid == 0 && a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);
  // All pages (pass 0); then the number of documents that begin before the share, and before its end.  Up to kThreads documents are
  // looked at once.
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    int64_t before = 0;
#pragma unroll 1
    for (int d0 = 0; d0 < nd; d0 += kThreads) {
      int st = 0, ln = 0;
      if (d0 + tid < nd) span(d0 + tid, st, ln);
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
        lo = (int64_t)sum * share / shares;
        hi = (int64_t)sum * (share + 1) / shares;
      }
      if (pass == 1 || only) {
        const unsigned below = __ballot_sync(0xffffffffu, d0 + tid < nd && before + first < lo);
        const unsigned below_end = __ballot_sync(0xffffffffu, d0 + tid < nd && (before + first < hi || share + 1 == shares));
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
      lo = before * share / shares;
      hi = before * (share + 1) / shares;
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
      sl2[c][x] = q.exponent_scale(a.scale, c, x);
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
    if (lane < n_docs) span(doc0 + lane, start, len);
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
    if (a.whole) {  // (one batch) a warp has some of the rows, a lane a document
      constexpr int kMine = kCols / kWarps;
      float e[kMine], top[kMine], z[kMine], mine = 0.f;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        float2 ml[kWarps];
        top[i] = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          ml[w] = s_ml[w][lane][warp + kWarps * i];  // ((-infinity, 0) of documents that are not there)
          top[i] = fmaxf(top[i], ml[w].x);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], off));
        const float ref = top[i] == -INFINITY ? 0.f : top[i];
        e[i] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) e[i] = fmaf(ml[w].y, ptx::ex2(ml[w].x - ref), e[i]);
        z[i] = e[i];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) z[i] += __shfl_xor_sync(0xffffffffu, z[i], off);
      }
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int r = warp + kWarps * i;
        const float p = z[i] != 0.f ? e[i] / z[i] : 0.f;  // (NaN stays NaN)
        if (r < GR && lane < nd) a.mass[(((int64_t)b * a.Nk + kvh) * GR + r) * nd + lane] = p;
        if (r < GR) mine += p;
      }
      s_mass[warp][lane] = mine;
      __syncthreads();
      if (warp == 0) {
        float total = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) total += s_mass[w][lane];
        s_total[lane] = total;
      }
      if (a.logits == nullptr) return;
      __syncwarp();
      if (a.Nk > 1) ptx::cluster_sync();
      float total = 0.f;
      if (kvh == 0 && warp == 0) {
        float of[kHeads];
#pragma unroll
        for (int c = 0; c < kHeads; ++c) of[c] = c == 0 ? s_total[lane] : c < a.Nk ? ptx::ld_cluster_f32(ptx::smem_u32(&s_total[lane]), c) : 0.f;
#pragma unroll
        for (int c = 0; c < kHeads; ++c) total += of[c];
        __syncwarp();
      }
      if (a.Nk > 1) ptx::cluster_arrive();
      if (kvh == 0 && warp == 0 && lane < nd) a.logits[(int64_t)b * nd + lane] = total * a.inv_count_temp;
      __syncwarp();
      if (a.Nk > 1) ptx::cluster_wait();  // nobody leaves while its sums are read
      return;
    }
    for (int i = tid; i < kDocs * kCols; i += kThreads) {
      const int doc = i % kDocs, r = row0 + i / kDocs;
      if (doc >= n_docs || r >= GR) continue;
      float2 ml = s_ml[0][doc][i / kDocs];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) ml = merged(ml, s_ml[w][doc][i / kDocs]);
      a.partial[(((int64_t)b * a.Nk + kvh) * GR + r) * nd + doc0 + doc] = ml;
    }
    __syncthreads();
  }
}

struct Split {
  int tiles, z;    // of 8 rows; CTAs of a KV head's rows
  int64_t shares;  // of a prompt's documents
  bool whole;
};
// Shares of a prompt's documents, at least a page (or short document) for each warp: a round of CTAs takes as long as its share, with about eight pages' time
// for beginning and end, and the kernel that merges what they find about twelve; a cluster that has all of a prompt needs none.  (In
// clusters and with the kernel: one prompt of 5 documents, 8 pages, 6.8 us and 8.1; 16 pages 8.6 and 8.4; 26 pages 10.3 and 9.1; 16
// prompts of 18 pages 10.6 and 11.5, of 46 pages 18.5 and 15.0.)
Split split_of(const brk_cache_score_params& p) {
  const int nd = p.M - 2, Nk = p.cache.Nk, rows = p.N / Nk * p.R, tiles = rows > 8 ? 2 : 1, z = (rows + 8 * tiles - 1) / (8 * tiles);
  Split r = {tiles, z, 1, false};
  const int64_t ctas = (int64_t)p.B * Nk * z, room = (tiles == 1 && p.dtype == BRK_BF16 ? 3 : 2) * (int64_t)std::max(1, sm_count());
  const int64_t pages = std::max(p.P, nd), most = std::min<int64_t>(nd, (pages + kWarps - 1) / kWarps);
  const bool may = z == 1 && nd <= kDocs && Nk <= kHeads;
  int64_t best = may ? (ctas + room - 1) / room * (pages + 8) : INT64_MAX;
  r.whole = may;
  for (int64_t round = 0; round <= 8; ++round) {  // (the most shares of so many rounds, and the fewest)
    const int64_t s = std::min(most, std::max<int64_t>(1, round * room / ctas));
    const int64_t cost = (ctas * s + room - 1) / room * ((pages + s - 1) / s + 8) + 12;
    if (cost < best) {
      best = cost;
      r.shares = s;
      r.whole = false;
    }
  }
  return r;
}

}  // namespace


size_t cache_scores_workspace(const brk_cache_score_params& p) {
  return split_of(p).whole ? 0 : (size_t)p.B * p.N * p.R * (p.M - 2) * sizeof(float2);
}

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
  const Split split = split_of(p);
  a.whole = split.whole;
  a.mass = p.doc_mass;
  a.logits = p.logits;
  a.inv_count_temp = 1.f / ((float)(p.N * p.R) * p.temperature);
  const int tiles = split.tiles;
  const dim3 grid = split.whole ? dim3(a.Nk, p.B) : dim3((unsigned)split.shares, p.B * a.Nk, split.z);
  auto run = [&](auto kern, std::atomic<bool>* configured) -> int {
    const int bytes = kWarps * kStages * (int)head_page_bytes(p.cache.D) / 2;
    int dev = 0;
    BRK_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
      BRK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      BRK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared));
      if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    return launch_dependent_clusters(a.whole ? a.Nk : 1, kern, grid, dim3(kThreads), bytes, st, a);
  };
  static std::atomic<bool> done[8][64] = {};
  auto of_head_dim = [&](auto d, std::atomic<bool>(*flags)[64]) -> int {
    constexpr int D = decltype(d)::value;
    if (p.dtype == BRK_F32) return tiles == 1 ? run(cache_scores_kernel<float, D, 1>, flags[0]) : run(cache_scores_kernel<float, D, 2>, flags[1]);
    return tiles == 1 ? run(cache_scores_kernel<__nv_bfloat16, D, 1>, flags[2]) : run(cache_scores_kernel<__nv_bfloat16, D, 2>, flags[3]);
  };
  const int rc = p.cache.D == 128 ? of_head_dim(std::integral_constant<int, 128>(), done) : of_head_dim(std::integral_constant<int, 64>(), done + 4);
  if (rc || a.whole) return rc;
  ScoreArgs m = {};
  m.partial = a.partial;
  m.mass = p.doc_mass;
  m.logits = p.logits;
  m.inv_count_temp = a.inv_count_temp;
  m.keep_nan = true;
  m.B = p.B; m.N = p.N; m.Nk = a.Nk; m.M = p.M; m.R = p.R;
  return doc_merge_launch(m, st);
}

}  // namespace brk
