// Document scores from the 4-bit cache: the signal rows against the held keys of every document.
//
// A warp takes a document (or a part of its pages, where there are few documents) for one KV head and up to 8 kTiles (head, signal
// row) pairs and keeps a running (maximum, sum) per pair; the pairs of a prompt's documents are merged by the kernel that
// merges those of doc_scores.  Bound by the read of the keys (72 bytes per token and KV head at head_dim 128).
#include <algorithm>
#include <atomic>

#include "cache_layout.cuh"
#include "score_args.cuh"
#include "tc_ptx.cuh"

namespace brk {
namespace {

using namespace cache;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 3;  // pages (their K parts) a warp has in shared memory
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
  int split;  // warps per document: 1 or kWarps
  float scale;
};

template <typename T, int D, int kTiles>
__global__ void __launch_bounds__(kThreads, kTiles == 1 && sizeof(T) == 2 ? 4 : 2) cache_scores_kernel(CacheScoreArgs a) {
  using L = Layout<D>;
  constexpr int kCols = 8 * kTiles;
  extern __shared__ __align__(16) unsigned char smem[];  // [kWarps][kStages][K part of a page]
  __shared__ float2 s_ml[kWarps][kCols];
  ptx::grid_dependency_wait();
  ptx::grid_dependency_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int b = blockIdx.y / a.Nk, kvh = blockIdx.y % a.Nk, row0 = blockIdx.z * kCols;
  const int G = a.N / a.Nk, GR = G * a.R, nd = a.M - 2;
  const int doc = (blockIdx.x * kWarps + warp) / a.split, part = warp % a.split;

  int start = 0, len = 0;
  if (doc < nd) {
    const int32_t *bs = a.blk_start + (int64_t)b * a.M, *bl = a.blk_len + (int64_t)b * a.M;
    start = bs[doc + 1];
    len = bl[doc + 1];
    if (span_is_bad(bs, bl, doc + 1, (int64_t)a.P * kPage) || len > a.max_block_len) {
      if (lane == 0 && a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);
      len = 0;
    }
  }
  const int page0 = start / kPage, n = len > 0 ? (start + len - 1) / kPage - page0 + 1 : 0;  // the document's pages

  unsigned char* const ring = smem + warp * kStages * L::kHalf;
  const unsigned char* const head = a.pages + (int64_t)kvh * L::kBytes;
  int ids = -1, ids0 = -32;  // page numbers of the pages ids0 .. ids0 + 31, one per lane
  auto page_of = [&](int i) {
    if (i >= ids0 + 32) {
      ids0 = i;
      ids = i + lane < n ? a.table[(int64_t)b * a.P + page0 + i + lane] : 0;
      if (__any_sync(0xffffffffu, ids < 0 || ids >= a.n_pages)) {
        if (lane == 0 && a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);
        if (ids >= a.n_pages) ids = -1;
      }
    }
    return __shfl_sync(0xffffffffu, ids, i - ids0);
  };
  uint32_t absent = 0;  // bit s: the page in stage s does not exist
  auto request = [&](int i, int stage) {
    if (i < n) {
      const int page = page_of(i);
      absent = page < 0 ? absent | (1u << stage) : absent & ~(1u << stage);
      if (page >= 0) {
        const unsigned char* src = head + (int64_t)page * a.Nk * L::kBytes;
        for (int x = lane * 16; x < L::kHalf; x += 512) cp_async16(ring + stage * L::kHalf + x, src + x);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages; ++s) request(part + s * a.split, s);

  QueryRows<T, D, kTiles> q;
  q.load([&](int c) -> const T* {
    const int r = row0 + c;
    if (r >= GR) return nullptr;
    return reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb + (int64_t)(kvh * G + r / a.R) * a.q.sh + (int64_t)(r % a.R) * a.q.ss;
  }, g, t);
  float sl2[kTiles][2], mx[kTiles][2], sum[kTiles][2];  // this lane's keys
#pragma unroll
  for (int c = 0; c < kTiles; ++c)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      sl2[c][x] = a.scale * kLog2e * q.unit[c][x];
      mx[c][x] = -INFINITY;
      sum[c][x] = 0.f;
    }
  int stage = 0;
  for (int i = part; i < n; i += a.split) {
    cp_async_wait<kStages - 1>();
    __syncwarp();
    if (!((absent >> stage) & 1)) {
      float s[kTiles][4][4];
      q.logits(ring + stage * L::kHalf, g, t, s);
      const int from = start - (page0 + i) * kPage, to = start + len - (page0 + i) * kPage;  // the document's tokens in this page
      if (from > 0 || to < kPage) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int key = 16 * k + 8 * y + g;
            if (key < from || key >= to) {
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
    __syncwarp();
    request(i + kStages * a.split, stage);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();
#pragma unroll
  for (int c = 0; c < kTiles; ++c)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float m = mx[c][x] * sl2[c][x], l = sum[c][x];
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, off), l2 = __shfl_xor_sync(0xffffffffu, l, off);
        const float top = fmaxf(m, m2), ref = top == -INFINITY ? 0.f : top;
        l = l * ptx::ex2(m - ref) + l2 * ptx::ex2(m2 - ref);
        m = top;
      }
      if (g == 0) s_ml[warp][8 * c + 2 * t + x] = make_float2(m, l);
    }
  if (a.split > 1) __syncthreads();
  else __syncwarp();
  if (doc >= nd || part != 0) return;
  for (int col = lane; col < kCols && row0 + col < GR; col += 32) {
    float2 ml = s_ml[warp][col];
    for (int w = 1; w < a.split; ++w) {
      const float2 x = s_ml[warp + w][col];
      const float top = fmaxf(ml.x, x.x), ref = top == -INFINITY ? 0.f : top;
      ml = make_float2(top, ml.y * ptx::ex2(ml.x - ref) + x.y * ptx::ex2(x.x - ref));
    }
    const int r = row0 + col;
    a.partial[(((int64_t)b * a.N + kvh * G + r / a.R) * a.R + r % a.R) * nd + doc] = ml;
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
  a.split = (int64_t)nd * p.B * a.Nk * z < 8 * (int64_t)std::max(1, sm_count()) || p.max_block_len > 16 * kPage ? kWarps : 1;
  const dim3 grid((nd * a.split + kWarps - 1) / kWarps, p.B * a.Nk, z);
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
  int rc;
  const bool f32 = p.dtype == BRK_F32;
  if (p.cache.D == 128) {
    if (f32) rc = tiles == 1 ? run(cache_scores_kernel<float, 128, 1>, done[0]) : run(cache_scores_kernel<float, 128, 2>, done[1]);
    else rc = tiles == 1 ? run(cache_scores_kernel<__nv_bfloat16, 128, 1>, done[2]) : run(cache_scores_kernel<__nv_bfloat16, 128, 2>, done[3]);
  } else {
    if (f32) rc = tiles == 1 ? run(cache_scores_kernel<float, 64, 1>, done[4]) : run(cache_scores_kernel<float, 64, 2>, done[5]);
    else rc = tiles == 1 ? run(cache_scores_kernel<__nv_bfloat16, 64, 1>, done[6]) : run(cache_scores_kernel<__nv_bfloat16, 64, 2>, done[7]);
  }
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
