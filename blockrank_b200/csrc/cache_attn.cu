// Attention of a prompt's last tokens over its pages of the 4-bit cache, and the join of its parts.
//
// out = sum_j softmax_j(scale q . k_j) v_j over the slots j that row i sees: those of all blocks at or before its own slot.
// Bound by the read of the cache (144 bytes per token and KV head at head_dim 128), with 72 % of the issue slots needed to keep up
// with it (counted from the source: 287 instructions per 16 keys and warp).
//
// A CTA takes a share of one prompt's pages for one KV head and up to 8 kTiles rows (a row: a query head of the group at one
// token).  Its warps take whole pages in turn and share nothing until the end: running maximum, sum and output of a warp
// stay in its registers, pages come through a ring of asynchronous copies of its own.  Both products have the cache as
// their 16-row operand and the rows as the 8-column one, because a decoding step has few rows: S^T = K Q^T, O^T = V^T P^T.
// P passes from the first to the second by one 8 x 8 transposition of packed pairs.
//
// P is not rounded to 8 bits: it goes in as two bf16 numbers (16 bits) next to bf16 inputs, three (all 24) next to fp32, and
// fp32 queries as three.  The held values are exact in bf16, so these are the only roundings in front of the 32-bit sums.
#include <algorithm>
#include <atomic>

#include "cache_layout.cuh"
#include "tc_ptx.cuh"

namespace brk {
namespace {

using namespace cache;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 2;        // pages a warp has in shared memory
constexpr int kShare = 512;       // pages a CTA takes at most
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
  float scale;
};

// rows of prompt b, or -1 if its spans or its number of rows are malformed (all threads of the CTA)
__device__ __forceinline__ int checked_rows(const CacheAttnArgs& a, int b) {
  const int32_t *start = a.blk_start + (int64_t)b * a.M, *len = a.blk_len + (int64_t)b * a.M;
  bool bad = false;
  for (int m = threadIdx.x; m < a.M; m += blockDim.x) bad |= span_is_bad(start, len, m, (int64_t)a.P * kPage);
  const int rows = a.q_len ? a.q_len[b] : a.Lq;
  bad |= rows < 0 || rows > a.Lq || rows > len[a.M - 1];
  return __syncthreads_or(bad) ? -1 : rows;
}

template <typename T, int D, int kTiles>
__global__ void __launch_bounds__(kThreads) cache_attn_kernel(CacheAttnArgs a) {
  using L = Layout<D>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kQ = kF32 ? 3 : 1, kP = kF32 ? 3 : 2;
  constexpr int kCols = 8 * kTiles;
  extern __shared__ __align__(16) unsigned char smem[];  // [kWarps][kStages][page]; at the end the warps' outputs
  __shared__ uint32_t s_mask[2 * kShare];                // which tokens of the CTA's pages lie in a block
  __shared__ int32_t s_page[kShare];
  __shared__ float2 s_ml[kWarps][kCols];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int share = blockIdx.x, b = blockIdx.y / a.Nk, kvh = blockIdx.y % a.Nk, row0 = blockIdx.z * kCols;
  const int G = a.N / a.Nk;
  ptx::grid_dependency_launch();
  ptx::grid_dependency_wait();  // (inputs of this call; the workspace of the one in front)
  const int checked = checked_rows(a, b), rows = max(checked, 0);
  if (checked < 0 && tid == 0 && a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);
  const int n_rows = min(rows * G - row0, kCols);  // of this CTA
  const int32_t *start = a.blk_start + (int64_t)b * a.M, *len = a.blk_len + (int64_t)b * a.M;
  const int first_slot = start[a.M - 1] + len[a.M - 1] - rows;  // of the prompt's row 0
  // this CTA's pages: an even share of those up to the last row's slot
  const int last_tok = n_rows > 0 ? (row0 + n_rows - 1) / G : -1;
  const int live = n_rows > 0 ? (first_slot + last_tok) / kPage + 1 : 0;
  const int per = max((live + a.shares - 1) / a.shares, min(live, kWarps));
  const int page0 = min(live, share * per), n = min(live, page0 + per) - page0;

  // ---- which tokens of these pages lie in a block ----
  for (int i = tid; i < 2 * n; i += kThreads) s_mask[i] = 0;
  __syncthreads();
  if (n > 0) {
    const int lo = page0 * kPage, hi = (page0 + n) * kPage;
    for (int m0 = warp * 32; m0 < a.M; m0 += kThreads) {
      const int m = m0 + lane;
      const int s = m < a.M ? start[m] : 0, e = m < a.M ? s + len[m] : 0;
      unsigned todo = __ballot_sync(0xffffffffu, max(s, lo) < min(e, hi));
      while (todo) {
        const int src = __ffs(todo) - 1;
        todo &= todo - 1;
        const int bs = max(__shfl_sync(0xffffffffu, s, src), lo) - lo, be = min(__shfl_sync(0xffffffffu, e, src), hi) - lo;
        for (int w = bs / 32 + lane; w * 32 < be; w += 32) {  // a word of 32 tokens per lane
          const int from = max(bs - w * 32, 0), to = min(be - w * 32, 32);
          atomicOr(&s_mask[w], (to == 32 ? ~0u : (1u << to) - 1) & (~0u << from));
        }
      }
    }
    __syncthreads();
    bool bad = false;
    for (int i = tid; i < n; i += kThreads) {
      int page = -1;
      if (s_mask[2 * i] | s_mask[2 * i + 1]) {
        page = a.table[(int64_t)b * a.P + page0 + i];
        if (page < 0 || page >= a.n_pages) {
          bad = true;
          page = -1;
        }
      }
      s_page[i] = page;
    }
    if (bad && a.status) atomicCAS(a.status, 0, kStatusBadCacheCall);
  }
  __syncthreads();

  // ---- the rows ----
  uint32_t q[kTiles][kQ][D / 32][2][2];
  int lim[kTiles][2];  // last slot that this lane's columns see
#pragma unroll
  for (int c = 0; c < kTiles; ++c) {
    const int r = row0 + 8 * c + g;
    const T* p = nullptr;
    if (8 * c + g < n_rows)
      p = reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb + (int64_t)(kvh * G + r % G) * a.q.sh + (int64_t)(r / G) * a.q.ss;
    load_query<D, kQ>(p, t, q[c]);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int col = 8 * c + 2 * t + x;
      lim[c][x] = col < n_rows ? first_slot + (row0 + col) / G : INT_MAX;
    }
  }
  const int first_lim = first_slot + row0 / G;  // the least of the CTA's rows
  const float sl2 = a.scale * kLog2e;
  float o[kTiles][L::kGroups][2][4] = {};
  float mx[kTiles][2], sum[kTiles][2];
#pragma unroll
  for (int c = 0; c < kTiles; ++c)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mx[c][x] = -INFINITY;
      sum[c][x] = 0.f;
    }

  unsigned char* const ring = smem + warp * kStages * L::kBytes;
  const unsigned char* const head = a.pages + (int64_t)kvh * L::kBytes + lane * 16;
  auto next = [&](int i) {  // the warp's next page with a token in it
    while (i < n && s_page[i] < 0) i += kWarps;
    return i;
  };
  auto request = [&](int i, int stage) {
    if (i < n) {
      const unsigned char* src = head + (int64_t)s_page[i] * a.Nk * L::kBytes;
      unsigned char* dst = ring + stage * L::kBytes + lane * 16;
#pragma unroll
      for (int x = 0; x < L::kBytes / 512; ++x) cp_async16(dst + 512 * x, src + 512 * x);
    }
    cp_async_commit();
  };
  int ahead = next(warp);
#pragma unroll
  for (int s = 0; s < kStages; ++s) {
    request(ahead, s);
    ahead = next(ahead + kWarps);
  }
  int stage = 0;
  for (int i = next(warp); i < n; i = next(i + kWarps)) {
    cp_async_wait<kStages - 1>();
    __syncwarp();
    const unsigned char* const page = ring + stage * L::kBytes;
    float s[kTiles][4][4];
    page_logits<D, kTiles, kQ>(page, q, g, t, s);

    // ---- softmax ----
    const int slot0 = (page0 + i) * kPage;
    const uint32_t m_lo = s_mask[2 * i], m_hi = s_mask[2 * i + 1];
    const bool whole = (m_lo & m_hi) == ~0u && slot0 + kPage - 1 <= first_lim;
    if (!whole) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int key = 16 * k + 8 * y + g;
          const bool in = ((key < 32 ? m_lo : m_hi) >> (key & 31)) & 1;
#pragma unroll
          for (int c = 0; c < kTiles; ++c)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              if (!in || slot0 + key > lim[c][x]) s[c][k][2 * y + x] = -INFINITY;
        }
    }
    float scale_o[kTiles][2];
    bool grown = false;
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float top = mx[c][x];
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, fmaxf(s[c][k][x], s[c][k][2 + x]));
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float ref = top == -INFINITY ? 0.f : top * sl2;
        scale_o[c][x] = ptx::ex2(mx[c][x] * sl2 - ref);  // (2^-inf = 0 in front of the first page)
        grown |= top > mx[c][x];
        mx[c][x] = top;
        sum[c][x] *= scale_o[c][x];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float p = ptx::ex2(fmaf(s[c][k][2 * y + x], sl2, -ref));
            s[c][k][2 * y + x] = p;
            sum[c][x] += p;
          }
      }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int j = 0; j < L::kGroups; ++j)
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[c][j][y][x] *= scale_o[c][x & 1];
    }

    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t pt[kTiles][2][kP];
#pragma unroll
      for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          split2<kP>(s[c][k][2 * y], s[c][k][2 * y + 1], pt[c][y]);
#pragma unroll
          for (int x = 0; x < kP; ++x) pt[c][y][x] = transpose8(pt[c][y][x]);
        }
      // pairs of tokens 16 k + 2 t (v[0]) and 16 k + 8 + 2 t (v[1]); words of the even token, then of the odd one
      uint32_t v[2][2 * (L::kGroups / 2)], sv[2][L::kGroups];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int tok = 16 * k + 8 * y + 2 * t;
        const unsigned char *pv = page + L::v_word(tok, g, 0), *ps = page + L::v_scale(tok, 0);
        if constexpr (D == 128) {
          *reinterpret_cast<uint4*>(v[y]) = *reinterpret_cast<const uint4*>(pv);
          *reinterpret_cast<uint4*>(sv[y]) = *reinterpret_cast<const uint4*>(ps);
        } else {
          *reinterpret_cast<uint2*>(v[y]) = *reinterpret_cast<const uint2*>(pv);
          *reinterpret_cast<uint2*>(sv[y]) = *reinterpret_cast<const uint2*>(ps);
        }
      }
      if (!whole) {
        // Values of tokens that no row sees are zeros: 0 x NaN would reach every row.  One that some rows see and others do
        // not is dealt with below.
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int tok = 16 * k + 8 * y + 2 * t;
          const uint32_t in = (tok < 32 ? m_lo : m_hi) >> (tok & 31);
          const uint32_t keep = ((in & 1) ? 0xFFFFu : 0u) | ((in & 2) ? 0xFFFF0000u : 0u);
#pragma unroll
          for (int j = 0; j < L::kGroups; ++j) sv[y][j] &= keep;
        }
        uint32_t nan = 0;  // (a scale of all ones in the exponent is NaN)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int j = 0; j < L::kGroups; ++j) nan |= __vcmpeq2(sv[y][j] & 0x7F807F80u, 0x7F807F80u);
        if (__any_sync(0xffffffffu, nan != 0)) {
          // A value that is NaN belongs to the rows that see it and to no other: out of the product, into their outputs.
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int j = 0; j < L::kGroups; ++j) {
              const uint32_t is = __vcmpeq2(sv[y][j] & 0x7F807F80u, 0x7F807F80u);
              sv[y][j] &= ~is;
              int earliest = INT_MAX;  // slot of the first such token of these 8
              const int at = slot0 + 16 * k + 8 * y + 2 * t;
              if (is & 0xFFFF0000u) earliest = at + 1;
              if (is & 0xFFFFu) earliest = at;
              earliest = min(earliest, __shfl_xor_sync(0xffffffffu, earliest, 1));
              earliest = min(earliest, __shfl_xor_sync(0xffffffffu, earliest, 2));
#pragma unroll
              for (int c = 0; c < kTiles; ++c)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                  if (earliest <= lim[c][x & 1]) o[c][j][0][x] = o[c][j][1][x] = NAN;
            }
        }
      }
#pragma unroll
      for (int w = 0; w < L::kGroups / 2; ++w) {
        // the four bytes of each token, shifted by bytes: codes 2 i and 2 i + 1 of both in bits 3..6 and 7..10 of their halves
        uint32_t x[2][4];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t even = v[y][w], odd = v[y][L::kGroups / 2 + w];
          x[y][0] = __byte_perm(even, odd, 0x5410);
          x[y][1] = __byte_perm(even, odd, 0x6521);
          x[y][2] = __byte_perm(even, odd, 0x7632);
          x[y][3] = __byte_perm(even, odd, 0x4703);
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int j = 2 * w + z;
          uint32_t c2[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) c2[y] = scale_offset(sv[y][j]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {  // channels 4 g + 2 u, 4 g + 2 u + 1 of group j
            const uint32_t e0 = held(x[0][2 * z + u], sv[0][j], c2[0]), e1 = held(x[0][2 * z + u] >> 4, sv[0][j], c2[0]);
            const uint32_t f0 = held(x[1][2 * z + u], sv[1][j], c2[1]), f1 = held(x[1][2 * z + u] >> 4, sv[1][j], c2[1]);
#pragma unroll
            for (int c = 0; c < kTiles; ++c)
#pragma unroll
              for (int p = 0; p < kP; ++p) mma(o[c][j][u], e0, e1, f0, f1, pt[c][0][p], pt[c][1][p]);
          }
        }
      }
    }
    __syncwarp();
    request(ahead, stage);
    ahead = next(ahead + kWarps);
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();

  // ---- the warps' parts ----
#pragma unroll
  for (int c = 0; c < kTiles; ++c)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) sum[c][x] += __shfl_xor_sync(0xffffffffu, sum[c][x], off);
      if (g == 0) s_ml[warp][8 * c + 2 * t + x] = make_float2(mx[c][x] * sl2, sum[c][x]);
    }
  __syncthreads();  // every page has been used
  float* const s_o = reinterpret_cast<float*>(smem);  // [kWarps][kCols][D]
#pragma unroll
  for (int c = 0; c < kTiles; ++c)
#pragma unroll
    for (int j = 0; j < L::kGroups; ++j)
#pragma unroll
      for (int x = 0; x < 2; ++x)
        *reinterpret_cast<float4*>(s_o + (warp * kCols + 8 * c + 2 * t + x) * D + 32 * j + 4 * g) =
            make_float4(o[c][j][0][x], o[c][j][0][2 + x], o[c][j][1][x], o[c][j][1][2 + x]);
  __syncthreads();
  for (int i = tid; i < kCols * (D / 4); i += kThreads) {
    const int col = i / (D / 4), d = i % (D / 4) * 4;
    const int r = row0 + col, tok = r / G, hd = kvh * G + r % G;
    if (tok >= a.Lq) break;
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < n_rows) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ml[w][col].x);
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = s_ml[w][col];
        const float f = ptx::ex2(ml.x - ref);
        const float4 x = *reinterpret_cast<const float4*>(s_o + (w * kCols + col) * D + d);
        l = fmaf(ml.y, f, l);
        acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
      }
    }
    const int64_t row = ((int64_t)b * a.N + hd) * a.Lq + tok;
    if (a.shares > 1) {
      if (col >= n_rows && checked >= 0) continue;  // (the join looks at q_len: a malformed prompt's rows get statistics, of nothing)
      if (n > 0) store4(a.part_o + (row * a.shares + share) * D + d, acc);
      if (d == 0) a.part_ml[row * a.shares + share] = make_float2(m, l);
    } else {
      const float inv = l != 0.f ? 1.f / l : 0.f;  // (a sum that is NaN stays one)
      store4(reinterpret_cast<T*>(a.o.ptr) + (int64_t)b * a.o.sb + (int64_t)hd * a.o.sh + (int64_t)tok * a.o.ss + d,
             make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      if (a.lse && d == 0) a.lse[row] = l != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
    }
  }
}

// One warp per row.  A share without pages has written its statistics and nothing else.
template <typename T, int D>
__global__ void __launch_bounds__(128) cache_join_kernel(CacheAttnArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);  // (b, head, token)
  ptx::grid_dependency_wait();
  if (row >= (int64_t)a.B * a.N * a.Lq) return;
  const int tok = (int)(row % a.Lq), hd = (int)(row / a.Lq % a.N), b = (int)(row / a.Lq / a.N);
  const int rows = a.q_len ? a.q_len[b] : a.Lq;
  constexpr int kPer = D / 32;
  float acc[kPer] = {}, l = 0.f, ref = 0.f;
  if (tok < rows) {
    const float2* ml = a.part_ml + row * a.shares;
    float m = -INFINITY;
    for (int c = lane; c < a.shares; c += 32) m = fmaxf(m, ml[c].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    ref = m == -INFINITY ? 0.f : m;
    for (int c = 0; c < a.shares; ++c) {
      const float2 x = ml[c];
      if (x.y == 0.f) continue;
      const float f = ptx::ex2(x.x - ref);
      l = fmaf(x.y, f, l);
      const float* p = a.part_o + (row * a.shares + c) * D + lane;
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] = fmaf(p[32 * i], f, acc[i]);
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  T* dst = reinterpret_cast<T*>(a.o.ptr) + (int64_t)b * a.o.sb + (int64_t)hd * a.o.sh + (int64_t)tok * a.o.ss + lane;
#pragma unroll
  for (int i = 0; i < kPer; ++i) Elem<T>::store(dst + 32 * i, acc[i] * inv);
  if (a.lse && lane == 0) a.lse[row] = l != 0.f ? (ref + log2f(l)) * kLn2 : -INFINITY;
}

// Rows of a CTA: 8 or 16.
int row_tiles(const brk_cache_attn_params& p) { return (int64_t)p.Lq * (p.N / p.cache.Nk) > 8 ? 2 : 1; }

// Shares of a prompt's pages: CTAs for every SM several times over, as long as a share has a page for each warp, and none
// beyond kShare pages.
int shares_of(const brk_cache_attn_params& p) {
  const int64_t tiles = ((int64_t)p.Lq * (p.N / p.cache.Nk) + 8 * row_tiles(p) - 1) / (8 * row_tiles(p));
  const int64_t ctas = (int64_t)p.B * p.cache.Nk * tiles;
  const int64_t want = (3 * (int64_t)std::max(1, sm_count()) + ctas - 1) / ctas;
  const int64_t most = (p.P + kWarps - 1) / kWarps, least = (p.P + kShare - 1) / kShare;
  return (int)std::max(least, std::min(want, most));
}

}  // namespace

size_t cache_attn_workspace(const brk_cache_attn_params& p) {
  const size_t n = shares_of(p);
  return n > 1 ? (size_t)p.B * p.N * p.Lq * n * (p.cache.D * sizeof(float) + sizeof(float2)) : 0;
}

int cache_attn_launch(const brk_cache_attn_params& p, void* ws, cudaStream_t st) {
  CacheAttnArgs a;
  a.pages = static_cast<const unsigned char*>(p.cache.pages);
  a.q = make_view(p.q);
  a.o = make_view(p.o);
  a.table = p.page_table;
  a.blk_start = p.blk_start;
  a.blk_len = p.blk_len;
  a.q_len = p.q_len;
  a.lse = p.lse;
  a.status = p.status;
  a.n_pages = p.cache.n_pages; a.B = p.B; a.N = p.N; a.Nk = p.cache.Nk; a.Lq = p.Lq; a.M = p.M; a.P = p.P;
  a.shares = shares_of(p);
  a.scale = p.scale;
  const size_t rows = (size_t)p.B * p.N * p.Lq;
  a.part_o = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * a.shares * p.cache.D);
  const int tiles = row_tiles(p);
  const int64_t z = ((int64_t)p.Lq * (p.N / a.Nk) + 8 * tiles - 1) / (8 * tiles);
  BRK_REQUIRE(z <= 65535, BRK_E_UNSUPPORTED, "Lq * N / Nk = %lld rows are too many for one call", (long long)p.Lq * (p.N / a.Nk));
  const dim3 grid(a.shares, p.B * a.Nk, (unsigned)z);
  auto run = [&](auto kern, std::atomic<bool>* configured) -> int {
    const int bytes = kWarps * kStages * (int)head_page_bytes(p.cache.D);
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
    if (f32) rc = tiles == 1 ? run(cache_attn_kernel<float, 128, 1>, done[0]) : run(cache_attn_kernel<float, 128, 2>, done[1]);
    else rc = tiles == 1 ? run(cache_attn_kernel<__nv_bfloat16, 128, 1>, done[2]) : run(cache_attn_kernel<__nv_bfloat16, 128, 2>, done[3]);
  } else {
    if (f32) rc = tiles == 1 ? run(cache_attn_kernel<float, 64, 1>, done[4]) : run(cache_attn_kernel<float, 64, 2>, done[5]);
    else rc = tiles == 1 ? run(cache_attn_kernel<__nv_bfloat16, 64, 1>, done[6]) : run(cache_attn_kernel<__nv_bfloat16, 64, 2>, done[7]);
  }
  if (rc || a.shares == 1) return rc;
  const dim3 joins((unsigned)((rows + 3) / 4)), block(128);
  if (p.cache.D == 128)
    return f32 ? launch_dependent(cache_join_kernel<float, 128>, joins, block, 0, st, a)
               : launch_dependent(cache_join_kernel<__nv_bfloat16, 128>, joins, block, 0, st, a);
  return f32 ? launch_dependent(cache_join_kernel<float, 64>, joins, block, 0, st, a)
             : launch_dependent(cache_join_kernel<__nv_bfloat16, 64>, joins, block, 0, st, a);
}

}  // namespace brk
