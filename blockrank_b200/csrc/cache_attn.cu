// Attention of a prompt's last tokens over its pages of the 4-bit cache, and the join of its parts.
//
// out = sum_j softmax_j(scale q . k_j) v_j over the slots j that row i sees: those of all blocks at or before its own slot.
// The floor is the read of the cache (144 bytes per token and KV head at head_dim 128).  Bound by latency: a page's products, softmax and
// unpacking are one chain in a warp, which two or three warps to a scheduler cover in part.  From registers alone, 12 warps to an SM, a
// scheduler takes 364 cycles for 16 keys (K 139, softmax 40, V 206 where they are timed one by one), which would be 7.1 TB/s; in the kernel it
// takes 507 (5.3 TB/s at 1,965 MHz: two contexts of twice the tokens take 57.2 us more), 287 of them with an instruction; the ALU pipe, the
// busiest unit, is at 52 %.  One row each of two contexts of 131,072 tokens, 32 heads on 8: 69 us, 4.4 TB/s, of which 12 are beginning, end and
// join (kept up, the board's 1000 W bring the clock to 1,820 MHz: 73.5 us); of 16 prompts of 100 documents (32 to 256 tokens) 81 us, 3.2 TB/s:
// some SMs have two CTAs and some three, and 21 % more slots are worked on than there are tokens, because a document's last page is taken
// whole; of one prompt of 5 documents 7.3 us, all of it latency.
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
#include <type_traits>

#include "cache_share.cuh"

namespace brk {
namespace {

using namespace cache;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kAtOnce = 128;      // pages of its share that a CTA knows of at a time
constexpr int kWorthwhile = 128;  // pages that are worth a share of their own where there are more than 64
constexpr int kParts = 3;         // K or V parts of pages that a warp has room for in shared memory: two K, one V
constexpr int kFewJoins = 4;      // rows per SM that are joined by a CTA each
constexpr int kCluster = 8;       // shares that a cluster joins, at most (fp32, 3 prompts of 20 documents: 8.0 us, joined by a kernel 8.6)

template <typename T, int kTiles>
constexpr int ctas_per_sm = kTiles == 1 && sizeof(T) == 2 ? 3 : 2;

// kTwice: up to 4 rows, each in columns c and c + 4: the higher 8 bits of P go into one, the rest into the other, and one MMA takes
// both.
// kLong: a share can have more than kAtOnce pages.  (The code for that costs the others a little: one row each of 16 prompts of 100 documents
// 81.4 us, without it 80.9; of 4 in fp32 40.7 and 40.0.)
template <typename T, int D, int kTiles, bool kTwice, bool kLong>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<T, kTiles>) cache_attn_kernel(CacheAttnArgs a) {
  using L = Layout<D>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kP = kF32 ? 3 : 2, kMmas = kTwice ? 1 : kP;
  constexpr int kCols = 8 * kTiles, kRows = kTwice ? 4 : kCols;
  extern __shared__ __align__(16) unsigned char smem[];  // [kWarps][kParts][part]; at the end the warps' outputs
  __shared__ uint32_t s_mask[2 * kAtOnce];               // which tokens of the CTA's pages lie in a block
  __shared__ int32_t s_page[kAtOnce];
  __shared__ Prompt<kThreads> s_prompt;
  __shared__ float2 s_ml[kWarps][kCols];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int share = blockIdx.x, b = blockIdx.y / a.Nk, kvh = blockIdx.y % a.Nk, row0 = blockIdx.z * kRows;
  const int G = a.N / a.Nk;
  ptx::grid_dependency_launch();
  ptx::grid_dependency_wait();  // (inputs of this call; the workspace of the one in front)

  typename QueryRows<T, D, kTiles>::Raw raw;
  const Share sh = find_share<kAtOnce>(a, b, row0, kRows, share, kWarps, s_prompt, s_mask, s_page, [&] {
    QueryRows<T, D, kTiles>::fetch([&](int c) -> const T* {  // (rows from q_len on among them: they are not used)
      const int r = row0 + (kTwice ? c & 3 : c);
      if (r >= a.Lq * G) return nullptr;
      return reinterpret_cast<const T*>(a.q.ptr) + (int64_t)b * a.q.sb + (int64_t)(kvh * G + r % G) * a.q.sh + (int64_t)(r / G) * a.q.ss;
    }, g, t, raw);
  });
  const int n_rows = sh.n_rows, first_slot = sh.first_slot;
  int page0 = sh.page0, n = kLong ? min(sh.n, kAtOnce) : sh.n;  // the pages at hand

  // Copies are requested in the order K0 K1 V0 K2 V1 K3 ..., each into the place of the part that has just been used.
  unsigned char* const ring = smem + warp * kParts * L::kHalf;
  const unsigned char* const head = a.pages + (int64_t)kvh * L::kBytes;
  auto next = [&](int i) {  // the warp's next page with a token in it
    while (i < n && s_page[i] < 0) i += kWarps;
    return i;
  };
  auto request = [&](int i, int half, int place) {
    if (i < n) {
      const unsigned char* src = head + (int64_t)s_page[i] * a.Nk * L::kBytes + half * L::kHalf + lane * 16;
      unsigned char* dst = ring + place * L::kHalf + lane * 16;
#pragma unroll
      for (int x = 0; x < L::kHalf; x += 512)
        if (x + 512 <= L::kHalf || lane * 16 < L::kHalf - x) cp_async16(dst + x, src + x);
    }
    cp_async_commit();
  };
  int i = next(warp), ahead = next(i + kWarps);  // the page in hand, and the one whose K is requested next
  auto begin = [&] {
    request(i, 0, 0);
    request(ahead, 0, 1);
    request(i, 1, 2);
  };
  begin();

  // ---- the rows ----
  QueryRows<T, D, kTiles> q;
  q.make(raw, g, t);
  int lim[kTiles][2];  // last slot that this lane's columns see
  float sl2[kTiles][2];
#pragma unroll
  for (int c = 0; c < kTiles; ++c)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int col = 8 * c + (kTwice ? 2 * (t & 1) : 2 * t) + x;
      lim[c][x] = col < n_rows ? first_slot + (row0 + col) / G : INT_MAX;
      sl2[c][x] = q.exponent_scale(a.scale, c, x);
    }
  const int first_lim = first_slot + row0 / G;  // the least of the CTA's rows
  const Codes codes = a.codes;
  float o[kTiles][L::kGroups][2][4] = {};
  float mx[kTiles][2], sum[kTiles][2];
#pragma unroll
  for (int c = 0; c < kTiles; ++c)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      mx[c][x] = -INFINITY;
      sum[c][x] = 0.f;
    }

  int place = 0;  // of the page's K
  for (;;) {
    while (i < n) {
      const int i1 = ahead;
      ahead = next(ahead + kWarps);
      cp_async_wait<2>();
      __syncwarp();
      const int slot0 = (page0 + i) * kPage;
      const uint32_t m_lo = s_mask[2 * i], m_hi = s_mask[2 * i + 1];
      const bool ragged = (m_lo & m_hi) != ~0u, late = slot0 + kPage - 1 > first_lim;  // tokens that no row sees, that some do not see
      float s[kTiles][4][4];
      q.logits(ring + place * L::kHalf, g, t, s);
      __syncwarp();
      request(ahead, 0, place);
      place ^= 1;

      // ---- softmax ----
      // (A page's last tokens are worked on whether they count or not: left out 16 at a time, with a branch each, two contexts of
      // 131,072 tokens took 77 us, not 69; with code of their own for pages that end early 16 prompts of 100 documents 100, not 87.)
      if (ragged) {
        const uint32_t lo = m_lo >> g, hi = m_hi >> g;  // this lane's keys: every eighth bit
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int y = 0; y < 2; ++y)
            if (!((k < 2 ? lo : hi) & (1u << (16 * (k & 1) + 8 * y)))) {
#pragma unroll
              for (int c = 0; c < kTiles; ++c) s[c][k][2 * y] = s[c][k][2 * y + 1] = -INFINITY;
            }
      }
      if (late) {
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int last = lim[c][x] - slot0 - g;
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int y = 0; y < 2; ++y)
                if (16 * k + 8 * y > last) s[c][k][2 * y + x] = -INFINITY;
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
          const float ref = top == -INFINITY ? 0.f : top * sl2[c][x];
          scale_o[c][x] = ptx::ex2(mx[c][x] * sl2[c][x] - ref);  // (2^-inf = 0 in front of the first page)
          grown |= top > mx[c][x];
          mx[c][x] = top;
          sum[c][x] *= scale_o[c][x];
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float p = ptx::ex2(fmaf(s[c][k][2 * y + x], sl2[c][x], -ref));
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
      cp_async_wait<1>();
      __syncwarp();
      const unsigned char* const page = ring + 2 * L::kHalf - L::kHalf;  // (the third part; offsets count from a page's beginning)
      // The tensor cores cut a sum off rather than round it, so in 32 bits a page has sums of its own.
      float fresh[kF32 ? kTiles : 1][L::kGroups][2][4] = {};
      auto& sums = [&]() -> float (&)[kTiles][L::kGroups][2][4] {
        if constexpr (kF32) return fresh;
        else return o;
      }();
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t pt[kTiles][2][kMmas];
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t piece[kP];
            split2<kP>(s[c][k][2 * y], s[c][k][2 * y + 1], piece);
            if constexpr (kTwice) {
              pt[c][y][0] = transpose8(t < 2 ? piece[0] : piece[1]);
            } else {
#pragma unroll
              for (int x = 0; x < kP; ++x) pt[c][y][x] = transpose8(piece[x]);
            }
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
        if (ragged) {  // values of tokens that no row sees are zeros: 0 x NaN would reach every row
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int tok = 16 * k + 8 * y + 2 * t;
            const uint32_t in = (tok < 32 ? m_lo : m_hi) >> (tok & 31);
            const uint32_t keep = ((in & 1) ? 0xFFFFu : 0u) | ((in & 2) ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int j = 0; j < L::kGroups; ++j) sv[y][j] &= keep;
          }
        }
        if (late) {
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
              const uint32_t e0 = held(codes, x[0][2 * z + u], sv[0][j], c2[0]), e1 = held(codes, x[0][2 * z + u] >> 4, sv[0][j], c2[0]);
              const uint32_t f0 = held(codes, x[1][2 * z + u], sv[1][j], c2[1]), f1 = held(codes, x[1][2 * z + u] >> 4, sv[1][j], c2[1]);
#pragma unroll
              for (int c = 0; c < kTiles; ++c)
#pragma unroll
                for (int p = kMmas - 1; p >= 0; --p) mma(sums[c][j][u], e0, e1, f0, f1, pt[c][0][p], pt[c][1][p]);
            }
          }
        }
      }
      if constexpr (kF32) {
#pragma unroll
        for (int c = 0; c < kTiles; ++c)
#pragma unroll
          for (int j = 0; j < L::kGroups; ++j)
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int x = 0; x < 4; ++x) o[c][j][y][x] += fresh[c][j][y][x];
      }
      __syncwarp();
      request(i1, 1, 2);
      i = i1;
    }
    cp_async_wait<0>();
    if (!kLong || page0 + n >= sh.page0 + sh.n) break;
    __syncthreads();  // every warp is through with these pages
    page0 += n;
    n = min(sh.page0 + sh.n - page0, kAtOnce);
    find_pages(a, lists_of(a, b), s_prompt, page0, n, tid, kThreads, s_mask, s_page);
    __syncthreads();
    i = next(warp);
    ahead = next(i + kWarps);
    place = 0;
    begin();
  }

  // ---- the warps' parts ----
#pragma unroll
  for (int c = 0; c < kTiles; ++c)
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) sum[c][x] += __shfl_xor_sync(0xffffffffu, sum[c][x], off);
      if (g == 0) s_ml[warp][8 * c + 2 * t + x] = make_float2(mx[c][x] * sl2[c][x], sum[c][x]);
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
  // the CTA's statistics and output of column `col`, channels d .. d + 3
  auto part = [&](int col, int d, float& m, float& l, float4& acc) {
    m = -INFINITY;
    l = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, s_ml[w][col].x);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = s_ml[w][col];
      const float f = ptx::ex2(ml.x - ref);
      float4 x = *reinterpret_cast<const float4*>(s_o + (w * kCols + col) * D + d);
      if constexpr (kTwice) {
        const float4 y = *reinterpret_cast<const float4*>(s_o + (w * kCols + col + 4) * D + d);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
      l = fmaf(ml.y, f, l);
      acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
    }
  };
  auto write = [&](int tok, int hd, int d, float m, float l, float4 acc) {
    const float inv = l != 0.f ? 1.f / l : 0.f;  // (a sum that is NaN stays one)
    store4(reinterpret_cast<T*>(a.o.ptr) + (int64_t)b * a.o.sb + (int64_t)hd * a.o.sh + (int64_t)tok * a.o.ss + d,
           make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    if (a.lse && d == 0) a.lse[((int64_t)b * a.N + hd) * a.Lq + tok] = l != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
  };
  float* const s_part = s_o + kWarps * kCols * D;  // [kRows][D], then the rows' statistics: what the cluster's other CTAs read
  for (int i = tid; i < kRows * (D / 4); i += kThreads) {
    const int col = i / (D / 4), d = i % (D / 4) * 4;
    const int r = row0 + col, tok = r / G, hd = kvh * G + r % G;
    if (tok >= a.Lq) break;
    float m, l;
    float4 acc;
    part(col, d, m, l, acc);
    if (col >= n_rows) {
      m = -INFINITY;
      l = 0.f;
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (a.cluster) {
      *reinterpret_cast<float4*>(s_part + col * D + d) = acc;
      if (d == 0) reinterpret_cast<float2*>(s_part + kRows * D)[col] = make_float2(m, l);
    } else if (a.shares > 1) {
      if (col >= n_rows && !sh.bad) continue;  // (the join looks at q_len: a malformed prompt's rows get statistics, of nothing)
      const int64_t row = ((int64_t)b * a.N + hd) * a.Lq + tok;
      if (sh.n > 0) store4(a.part_o + (row * a.shares + share) * D + d, acc);
      if (d == 0) a.part_ml[row * a.shares + share] = make_float2(m, l);
    } else {
      write(tok, hd, d, m, l, acc);
    }
  }
  if (!a.cluster) return;
  __syncwarp();  // (at head_dim 64 a warp has pieces of two rows, of which only one may exist)
  ptx::cluster_sync();
  // Every CTA joins some of the rows' pieces of 4 channels: at most kPieces to a thread.
  constexpr int kPieces = (kRows * (D / 4) / 2 + kThreads - 1) / kThreads;
  float4 acc[kPieces];
  float m[kPieces], l[kPieces];
#pragma unroll
  for (int n = 0; n < kPieces; ++n) {
    const int i = (tid + n * kThreads) * a.shares + share;
    if (i >= kRows * (D / 4)) break;
    const int col = i / (D / 4), d = i % (D / 4) * 4;
    const uint32_t at_ml = ptx::smem_u32(reinterpret_cast<float2*>(s_part + kRows * D) + col), at_o = ptx::smem_u32(s_part + col * D + d);
    float2 ml[kCluster];
    float4 x[kCluster];
    m[n] = -INFINITY;
    l[n] = 0.f;
    acc[n] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int c = 0; c < kCluster; ++c) {
      ml[c] = make_float2(-INFINITY, 0.f);
      x[c] = acc[n];
      if (c < a.shares) {
        ml[c] = ptx::ld_cluster_f32x2(at_ml, c);
        x[c] = ptx::ld_cluster_f32x4(at_o, c);
      }
    }
#pragma unroll
    for (int c = 0; c < kCluster; ++c) m[n] = fmaxf(m[n], ml[c].x);
    const float ref = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
    for (int c = 0; c < kCluster; ++c) {
      const float f = ptx::ex2(ml[c].x - ref);
      l[n] = fmaf(ml[c].y, f, l[n]);
      acc[n].x = fmaf(x[c].x, f, acc[n].x); acc[n].y = fmaf(x[c].y, f, acc[n].y); acc[n].z = fmaf(x[c].z, f, acc[n].z); acc[n].w = fmaf(x[c].w, f, acc[n].w);
    }
  }
  __syncwarp();
  ptx::cluster_arrive();  // (this CTA has read what it needs)
#pragma unroll
  for (int n = 0; n < kPieces; ++n) {
    const int i = (tid + n * kThreads) * a.shares + share, col = i / (D / 4), d = i % (D / 4) * 4;
    const int r = row0 + col, tok = r / G;
    if (i >= kRows * (D / 4) || tok >= a.Lq) break;
    write(tok, kvh * G + r % G, d, m[n], l[n], acc[n]);
  }
  __syncwarp();
  ptx::cluster_wait();  // nobody leaves while its part is read
}

// One CTA per row; D / 4 threads read a share's part, 4 channels each.  A share without pages has written its statistics alone.
// Bound by latency: a thread's first parts are requested together with the statistics.
template <typename T, int D>
__global__ void __launch_bounds__(128) cache_join_kernel(CacheAttnArgs a) {
  constexpr int kLanes = D / 4, kAtOnce = 128 / kLanes, kHeld = 4;
  __shared__ float4 s_acc[128];
  const int tid = threadIdx.x, lane = tid & 31, sub = tid / kLanes, d = tid % kLanes * 4;
  const int64_t row = blockIdx.x;  // (b, head, token)
  ptx::grid_dependency_wait();
  const int tok = (int)(row % a.Lq), hd = (int)(row / a.Lq % a.N), b = (int)(row / a.Lq / a.N);
  const int rows = a.q_len ? a.q_len[b] : a.Lq;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f, ref = 0.f;
  if (tok < rows) {
    const float2* const ml = a.part_ml + row * a.shares;
    const float* const part = a.part_o + row * a.shares * D + d;
    float4 held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (sub + i * kAtOnce < a.shares) held[i] = load4(part + (int64_t)(sub + i * kAtOnce) * D);
    float m = -INFINITY;
    for (int c = lane; c < a.shares; c += 32) m = fmaxf(m, ml[c].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    ref = m == -INFINITY ? 0.f : m;
    for (int c = lane; c < a.shares; c += 32) l = fmaf(ml[c].y, ptx::ex2(ml[c].x - ref), l);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    auto add = [&](int c, float4 x) {
      const float2 w = ml[c];
      if (w.y == 0.f) return;
      const float f = ptx::ex2(w.x - ref);
      acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y); acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (sub + i * kAtOnce < a.shares) add(sub + i * kAtOnce, held[i]);
    for (int c = sub + kHeld * kAtOnce; c < a.shares; c += kAtOnce) add(c, load4(part + (int64_t)c * D));
  }
  s_acc[tid] = acc;
  __syncthreads();
  if (sub != 0) return;
#pragma unroll
  for (int i = 1; i < kAtOnce; ++i) {
    const float4 x = s_acc[tid + i * kLanes];
    acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
  store4(reinterpret_cast<T*>(a.o.ptr) + (int64_t)b * a.o.sb + (int64_t)hd * a.o.sh + (int64_t)tok * a.o.ss + d,
         make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  if (a.lse && tid == 0) a.lse[row] = l != 0.f ? (ref + log2f(l)) * kLn2 : -INFINITY;
}

// The same for many rows: D / 4 threads a row, which share nothing; 8 parts at a time.  (A call of 18,432 rows in two parts 27.2 us, with a
// CTA to a row 42.2; 6,144 rows in nine 88.6 and 93.8; 288 rows 28.1 and 27.6.)
template <typename T, int D>
__global__ void __launch_bounds__(128) cache_join_rows_kernel(CacheAttnArgs a, int64_t n_rows) {
  constexpr int kLanes = D / 4, kHeld = 8;
  const int lane = threadIdx.x % kLanes, d = lane * 4;
  const int64_t at = (int64_t)blockIdx.x * (128 / kLanes) + threadIdx.x / kLanes, row = min(at, n_rows - 1);
  ptx::grid_dependency_wait();
  const int tok = (int)(row % a.Lq), hd = (int)(row / a.Lq % a.N), b = (int)(row / a.Lq / a.N);
  const bool there = tok < (a.q_len ? a.q_len[b] : a.Lq);
  const float2* const ml = a.part_ml + row * a.shares;
  const float* const part = a.part_o + row * a.shares * D + d;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f, m = -INFINITY;
  for (int c0 = 0; c0 < (there ? a.shares : 0); c0 += kHeld) {
    float2 w[kHeld];
    float4 x[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const bool on = c0 + i < a.shares;
      w[i] = on ? ml[c0 + i] : make_float2(-INFINITY, 0.f);
      x[i] = on ? load4(part + (int64_t)(c0 + i) * D) : acc;
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) top = fmaxf(top, w[i].x);
    const float ref = top == -INFINITY ? 0.f : top, old = ptx::ex2(m - ref);
    m = top;
    l *= old;
    acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      if (w[i].y == 0.f) continue;  // (a share without pages has written its statistics alone)
      const float f = ptx::ex2(w[i].x - ref);
      l = fmaf(w[i].y, f, l);
      acc.x = fmaf(x[i].x, f, acc.x); acc.y = fmaf(x[i].y, f, acc.y); acc.z = fmaf(x[i].z, f, acc.z); acc.w = fmaf(x[i].w, f, acc.w);
    }
  }
  if (at >= n_rows) return;
  const float inv = l != 0.f ? 1.f / l : 0.f;
  store4(reinterpret_cast<T*>(a.o.ptr) + (int64_t)b * a.o.sb + (int64_t)hd * a.o.sh + (int64_t)tok * a.o.ss + d,
         make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  if (a.lse && lane == 0) a.lse[row] = l != 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// Which kernel, how many rows to a CTA, into how many shares a prompt's pages go.
struct Plan {
  bool many;  // the tcgen05 kernel
  int rows;   // of a CTA
  int64_t groups, shares, cost;
  // its cluster joins the parts of a prompt's shares; otherwise a kernel does
  bool cluster() const { return shares > 1 && shares <= kCluster && !many; }
};

// Shares: a round of CTAs takes as long as its share, with about six pages' time for beginning and end (in the tcgen05 kernel four); what is
// left over of the SMs in the last round is lost.  Clusters find fewer places: each group of SMs that one cannot leave has up to s - 1 too few
// for another (of 296 places 296 for clusters of 2, 279 of 3, 264 of 8; of 444 444, 426 and 384; ten groups assumed here are more).  Taken for
// 296, 288 CTAs in clusters of 3 took 53 us, where 256 in clusters of 2 took 38.
// There are never more than eight rounds of CTAs that have shares, so the parts that a kernel joins are those of 8 x 148 CTAs of the tcgen05
// kernel at most (256 rows each: 158 MB at head_dim 128), however long the call.
Plan plan_with(const brk_cache_attn_params& p, bool many, int per_cta) {
  const int64_t rows = (int64_t)p.Lq * (p.N / p.cache.Nk), groups = (rows + per_cta - 1) / per_cta;
  const int per_sm = many ? 1 : p.dtype == BRK_BF16 && per_cta <= 8 ? 3 : 2, sms = sm_count();
  const int64_t ctas = (int64_t)p.B * p.cache.Nk * groups, room = per_sm * (int64_t)(sms > 0 ? sms : 148);  // (workspaces are asked for without a device too)
  const int64_t pages = many ? 2 : kWarps;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(std::max(64, p.P / kWorthwhile), (p.P + pages - 1) / pages));
  Plan best = {many, per_cta, groups, 1, INT64_MAX};
  auto consider = [&](int64_t s) {
    const bool cluster = s > 1 && s <= kCluster && !many;
    const int64_t places = cluster ? std::max<int64_t>(s, s == 2 ? room : room - 10 * (s - 1)) : room;
    const int64_t join = s == 1 ? 0 : many ? 3 + s / 8 : cluster ? 2 : 6 + s / 8;
    const int64_t cost = (ctas * s + places - 1) / places * ((p.P + s - 1) / s + (many ? 4 : 6)) + join;
    if (cost < best.cost) {
      best.cost = cost;
      best.shares = s;
    }
  };
  for (int64_t round = 0; round <= 8; ++round) {  // (the most shares of so many rounds, and the fewest)
    const int64_t s = std::min(most, std::max<int64_t>(1, round * room / ctas));
    consider(s);
    if (s > 1) consider(s - 1);
    if (s == most) break;
  }
  return best;
}

// Rows of a CTA: 4 (bf16), 8 or 16; 256 in the tcgen05 kernel.  Fewer columns than rows would read the cache twice; 4 rows stand in 8 columns
// so that one product takes both parts of P.  (fp32 at head_dim 128 has no registers for 16: 2 prompts of 100 documents, 16 rows
// 47 us, with 8 to a CTA 36; 64 rows 135 and 113.  At head_dim 64 32 rows 35 and 42, 16 rows 23 and 24.)
// Of more than 16 rows in bf16 each kernel's cost is compared: a page takes 0.93 us (head_dim 64: 0.7) here and 1 us there, 1.45 for
// more than 128 rows, and there are 5 us more in front and behind.  (One prompt of 2 documents of 128 tokens, 36 rows: 9.0 us here,
// 14.1 there; of 100 documents 28.1 and 27.7, with 128 rows 55 and 29.  16 prompts of 2 documents, 36 rows 19.0 and 14.7.)
Plan plan_of(const brk_cache_attn_params& p) {
  const int64_t rows = (int64_t)p.Lq * (p.N / p.cache.Nk);
  if (p.dtype == BRK_F32) return plan_with(p, false, rows <= 8 || p.cache.D == 128 ? 8 : 16);
  const Plan few = plan_with(p, false, rows <= 4 ? 4 : rows <= 8 ? 8 : 16);
  if (rows <= 16) return few;
  const Plan many = plan_with(p, true, 256);
  return few.cost * (p.cache.D == 128 ? 93 : 70) <= many.cost * (rows > 128 ? 145 : 100) + 500 ? few : many;
}

}  // namespace

size_t cache_attn_workspace(const brk_cache_attn_params& p) {
  const Plan plan = plan_of(p);
  return plan.shares > 1 && !plan.cluster() ? (size_t)p.B * p.N * p.Lq * plan.shares * (p.cache.D * sizeof(float) + sizeof(float2)) : 0;
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
  const Plan plan = plan_of(p);
  a.shares = (int)plan.shares;
  a.scale = p.scale;
  a.cluster = plan.cluster();
  const size_t rows = (size_t)p.B * p.N * p.Lq;
  a.part_o = static_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + rows * a.shares * p.cache.D);
  BRK_REQUIRE(plan.groups <= 65535, BRK_E_UNSUPPORTED, "Lq * N / Nk = %lld rows are too many for one call", (long long)p.Lq * (p.N / a.Nk));
  const dim3 grid(a.shares, p.B * a.Nk, (unsigned)plan.groups);
  auto run = [&](auto kern, std::atomic<bool>* configured) -> int {
    const int bytes = kWarps * kParts * (int)head_page_bytes(p.cache.D) / 2;
    int dev = 0;
    BRK_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
      BRK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      BRK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, (int)cudaSharedmemCarveoutMaxShared));
      if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    return launch_dependent_clusters(a.cluster ? a.shares : 1, kern, grid, dim3(kThreads), bytes, st, a);
  };
  static std::atomic<bool> done[20][64] = {};
  const bool f32 = p.dtype == BRK_F32;
  auto of = [&](auto d, auto is_long, std::atomic<bool>(*flags)[64]) -> int {
    constexpr int D = decltype(d)::value;
    constexpr bool kLong = decltype(is_long)::value;
    if constexpr (D == 64)
      if (f32 && plan.rows == 16) return run(cache_attn_kernel<float, D, 2, false, kLong>, flags[1]);
    if (f32) return run(cache_attn_kernel<float, D, 1, false, kLong>, flags[0]);
    if (plan.rows == 4) return run(cache_attn_kernel<__nv_bfloat16, D, 1, true, kLong>, flags[2]);
    return plan.rows == 8 ? run(cache_attn_kernel<__nv_bfloat16, D, 1, false, kLong>, flags[3])
                          : run(cache_attn_kernel<__nv_bfloat16, D, 2, false, kLong>, flags[4]);
  };
  auto of_head_dim = [&](auto d, std::atomic<bool>(*flags)[64]) -> int {
    return (p.P + a.shares - 1) / a.shares > kAtOnce ? of(d, std::true_type(), flags + 5) : of(d, std::false_type(), flags);
  };
  const int rc = plan.many ? cache_attn_tc_launch(a, p.cache.D, st)
                 : p.cache.D == 128 ? of_head_dim(std::integral_constant<int, 128>(), done)
                                    : of_head_dim(std::integral_constant<int, 64>(), done + 10);
  if (rc || a.shares == 1 || a.cluster) return rc;
  auto join = [&](auto d, auto t) -> int {
    constexpr int D = decltype(d)::value;
    using T = decltype(t);
    if (rows <= (size_t)kFewJoins * std::max(1, sm_count())) return launch_dependent(cache_join_kernel<T, D>, dim3((unsigned)rows), dim3(128), 0, st, a);
    const int per = 512 / D;  // rows of a CTA
    return launch_dependent(cache_join_rows_kernel<T, D>, dim3((unsigned)((rows + per - 1) / per)), dim3(128), 0, st, a, (int64_t)rows);
  };
  if (p.cache.D == 128) return f32 ? join(std::integral_constant<int, 128>(), float()) : join(std::integral_constant<int, 128>(), __nv_bfloat16());
  return f32 ? join(std::integral_constant<int, 64>(), float()) : join(std::integral_constant<int, 64>(), __nv_bfloat16());
}

}  // namespace brk
