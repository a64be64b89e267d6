// Attention of many rows (a whole query block) over the 4-bit cache, on the tcgen05 tensor cores; bf16.
//
// A CTA takes a share of one prompt's pages for one KV head and up to 256 rows (query heads of the group at one token after the other), two
// tiles of 128.  Per page: four warps bring the codes out of the cache and write n s, exact in bf16, as the K and V operands
// (128-byte swizzle); one thread issues S = Q K^T and O += P V per tile; a thread per row makes P from S in tensor memory, in two
// bf16 parts (16 bits) that take the place of the 64 logits.  S is held twice, K and V three times, so that a page's Q K^T runs while
// the softmax is at the page before and the next one is being unpacked.  With up to 128 rows both groups of softmax threads work on the
// one tile, at every other page each, and put their outputs together at the end.
//
// Channels stand in K and V in whatever order the codes come out in, without a permutation: Q's are brought into K's order once, O's
// columns are given their names as they are written.
//
// Bound by the chain that a page is for a softmax thread (S out of tensor memory, maximum, exponentials, P into it: 2,200 of a page's
// 2,350 cycles by clocks read inside, 45 tokens by 4 heads), which two such warps and one that unpacks to a scheduler cover in part.  Two
// tiles of 192 rows, 64 pages more to a CTA: 1.41 us a page, under the profiler 2,590 cycles, in which a scheduler has 1,385 instructions; ALU
// pipe 41 %, special functions 40 %, tensor pipe 56 %.  One tile: 1.0 us.  4 prompts of 100 documents of 160 tokens, up to 45 tokens by 4 heads: 104 us, of
// which a CTA has 18,000 cycles in front of its pages and behind them.  On the way there:
// products issued in a loop 131 us, unrolled 125; Q by asynchronous copies 120.6; one tile by both groups, outputs through
// shared memory 117; no permutations 110; of a page that ends in its first half only that half 107, the parts joined
// by more rows to a CTA 105.  (Q in tensor memory, one S to a tile: 124 where this took 125.)
//
// Tensor memory: per tile S (64 columns) twice and O (D columns).  Shared memory at head_dim 128: Q 64 KB, K and V 3 x 32 KB, codes on
// their way 4 x 12 KB.
// Every wait is bounded (ptx::BoundedWaits).
#include <algorithm>
#include <atomic>

#include "cache_share.cuh"

namespace brk {
namespace {

using namespace cache;

constexpr int kAtOnce = 256;               // pages of its share that a CTA knows of at a time
constexpr int kTile = 128;                 // rows of a tile
constexpr int kSoftWarps = 8, kUnpackWarps = 4;
constexpr int kMmaWarp = kSoftWarps + kUnpackWarps;
constexpr int kThreads = 32 * (kMmaWarp + 1);
constexpr int kBufs = 3;
constexpr int kAhead = 4;                  // pages whose codes are on their way
constexpr int kTmemCols = 512, kTileCols = 256, kColO = 128;
constexpr float kLazy = 8.f;               // O is brought in line when the reference moves by more than 2^8
constexpr int kWaitBudget = 1 << 18;
// Barriers.  S, P and O have two per tile, for even and odd pages: by the time that a page's S is there only the page before last is
// sure to have reached O, so a single one's parity would not tell the last two pages apart.
constexpr int kKVFull = 0, kKVEmpty = kKVFull + kBufs, kSFull = kKVEmpty + kBufs, kPFull = kSFull + 4, kODone = kPFull + 4, kNumBars = kODone + 4;

template <int D>
struct Smem {
  static constexpr int kQChunk = kTile * 128, kQ = kTile * D * 2;   // 64 channels of a tile; a tile
  static constexpr int kChunk = kPage * 128, kHalf = kPage * D * 2; // 64 channels of a page's K (or V); all of it
  // What an unpacking thread copies of a page, every piece in a cell of its own: K words and V words twice, V scales; K scales twice.
  static constexpr int kCell = D / 8, kScales = D / 16, kThread = 5 * kCell + 2 * kScales, kStage = kThread * 32 * kUnpackWarps;
  static constexpr int kKV = 2 * kQ, kCodes = kKV + kBufs * 2 * kHalf, kBars = kCodes + kAhead * kStage, kBytes = kBars + kNumBars * 8 + 16;
};

template <int kBytes>
__device__ __forceinline__ void cp_async(void* dst, const void* src) {
  const uint32_t d = ptx::smem_u32(dst);
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(kBytes) : "memory");
}
// 16 bytes, or zeros
__device__ __forceinline__ void cp_async_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t low_part(uint32_t hi, float x, float y) { return pack_bf16(x - bf_lo(hi), y - bf_hi(hi)); }

// kLong: a share can have more than kAtOnce pages.  (The code for that costs the others something: query blocks of 4 prompts of 100
// documents 108 us, without it 104.)
template <int D, bool kLong>
__global__ void __launch_bounds__(kThreads, 1) cache_attn_tc_kernel(CacheAttnArgs a) {
  using L = Layout<D>;
  using SM = Smem<D>;
  constexpr int kG = L::kGroups;
  extern __shared__ unsigned char smem_raw[];
  __shared__ uint32_t s_mask[2 * kAtOnce];
  __shared__ int32_t s_page[kAtOnce];
  __shared__ Prompt<kThreads> s_prompt;
  // The pages with a token in a block, in order, are numbered over the whole share: number k is page s_list[k % kAtOnce] of those at hand,
  // which begin with entry s_page0 of the page table and end with page s_known - 1.
  __shared__ int s_list[kAtOnce], s_known, s_page0;
  __shared__ bool s_more;  // there are entries behind them
  __shared__ uint32_t s_nan[kBufs][kG][2];  // pages that some rows see in part: tokens whose value is NaN, by group
  unsigned char* const smem = smem_raw + ((1024u - (ptx::smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sbase = ptx::smem_u32(smem);
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(smem + SM::kBars + kNumBars * 8);
  auto bar = [&](int i) { return sbase + SM::kBars + (uint32_t)i * 8u; };

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int share = blockIdx.x, b = blockIdx.y / a.Nk, kvh = blockIdx.y % a.Nk, row0 = blockIdx.z * 2 * kTile;
  const int G = a.N / a.Nk;
  if (tid == 0) {
    for (int i = 0; i < kNumBars; ++i)
      ptx::mbar_init(bar(i), i < kKVEmpty || (i >= kPFull && i < kODone) ? 4u : 1u);  // (by the warps that write K and V, or P)
    ptx::fence_barrier_init();
  }
  if (warp == kMmaWarp) {
    __syncwarp();
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::grid_dependency_launch();
  ptx::grid_dependency_wait();
  constexpr int kQUnits = D / 8, kQStep = kThreads / kQUnits;  // 16 bytes of a row to a thread
  const int q_unit = tid % kQUnits;
  auto q_place = [&](int rr) {
    return smem + (rr / kTile) * SM::kQ + (q_unit >> 3) * SM::kQChunk + (rr % kTile) * 128 + (((q_unit & 7) ^ (rr & 7)) << 4);
  };
  const Share sh = find_share<kAtOnce>(a, b, row0, 2 * kTile, share, 1, s_prompt, s_mask, s_page, [&] {
    // Q as the K-major A operand: rows of 128 bytes, their 16-byte units swizzled
    const __nv_bfloat16* const q = reinterpret_cast<const __nv_bfloat16*>(a.q.ptr);
    const int step_tok = kQStep / G, step_head = kQStep % G;
    int tok = (row0 + tid / kQUnits) / G, head = (row0 + tid / kQUnits) % G;
#pragma unroll 1
    for (int rr = tid / kQUnits; rr < 2 * kTile; rr += kQStep) {
      const bool there = tok < a.Lq;
      cp_async_or_zero(ptx::smem_u32(q_place(rr)),
                       there ? q + (int64_t)b * a.q.sb + (int64_t)(kvh * G + head) * a.q.sh + (int64_t)tok * a.q.ss + 8 * q_unit : q, there);
      tok += step_tok;
      head += step_head;
      if (head >= G) {
        head -= G;
        ++tok;
      }
    }
    cp_async_commit();
  });
  auto place = [](int k) { return kLong ? k & (kAtOnce - 1) : k; };
  auto make_list = [&](int page0, int known) {  // by a warp
    const int n = kLong ? min(sh.page0 + sh.n - page0, kAtOnce) : sh.n;
    for (int i = lane; i - lane < n; i += 32) {
      const bool there = i < n && s_page[i] >= 0;
      const unsigned all = __ballot_sync(0xffffffffu, there);
      if (there) s_list[place(known + __popc(all & ((1u << lane) - 1)))] = i;
      known += __popc(all);
    }
    if (lane == 0) {
      s_known = known;
      s_page0 = page0;
      s_more = page0 + n < sh.page0 + sh.n;
    }
  };
  if (warp == 0) make_list(sh.page0, 0);
  cp_async_wait<0>();
#pragma unroll 2
  for (int rr = tid / kQUnits; rr < 2 * kTile; rr += kQStep) {  // (what this thread has copied) channels in the order of K's
    uint4* const p = reinterpret_cast<uint4*>(q_place(rr));
    const uint4 x = *p;
    *p = make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
  }
  ptx::fence_proxy_async_smem();
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const bool split = sh.n_rows <= kTile;  // one tile: the softmax groups take its pages in turn
  const int first_lim = sh.first_slot + row0 / G;  // the last slot that the CTA's first row sees
  ptx::BoundedWaits waits(kWaitBudget);
  auto wait = [&](int i, uint32_t parity) { waits(bar(i), parity & 1u, 1); };
  // When all that is known of has been worked on, the warps that unpack look at the next kAtOnce entries, between two of these.
  auto meet = [] {
    __syncwarp();
    asm volatile("bar.sync 3, %0;" ::"n"(kThreads) : "memory");
  };
  auto unpackers_meet = [] {
    __syncwarp();
    asm volatile("bar.sync 1, 128;" ::: "memory");
  };

  if (warp < kSoftWarps) {
    // =============================== softmax: a thread per row ===========================================
    const int x = warp >> 2, rr = tid & (kTile - 1);
    int r = row0 + (split ? rr : tid);  // the thread's row
    bool there = r - row0 < sh.n_rows;
    const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)x * kTileCols;
    const int lim = sh.first_slot + r / G;
    const float sl2 = a.scale * kLog2e;
    float m_run = -INFINITY, l_run = 0.f;
    unsigned poison = 0;  // groups of channels in which this row has seen NaN
    int pages = 0;  // that this group has worked on
#pragma unroll 1
    for (;;) {
      const int to = split ? (s_known + 1 - x) / 2 : s_known, page0 = kLong ? s_page0 : sh.page0;
#pragma unroll 1
      for (; pages < to; ++pages) {
        const int j = pages;
        const int k = split ? 2 * j + x : j, i = s_list[place(k)], slot0 = (page0 + i) * kPage;
        unsigned v0 = s_mask[2 * i], v1 = s_mask[2 * i + 1];
        const uint32_t tm_s = tm + (uint32_t)(j & 1) * 64;
        const bool late = slot0 + kPage - 1 > first_lim;
        wait(kSFull + 2 * x + (j & 1), j >> 1);
        ptx::tc_fence_after_sync();
        __syncwarp();
        const bool two = v1 != 0;
        uint32_t sr[2][32];
        ptx::tmem_ld32(tm_s, sr[0]);
        if (two) ptx::tmem_ld32(tm_s + 32, sr[1]);
        ptx::tmem_wait_ld(sr[0]);
        if (two) ptx::tmem_wait_ld(sr[1]);
        if (late || (v0 & v1) != ~0u) {  // (warp-uniform)
          if (late) {
            const int n = there ? max(0, min(64, lim - slot0 + 1)) : 64;
            v0 &= n >= 32 ? ~0u : (1u << n) - 1u;
            v1 &= n >= 64 ? ~0u : n > 32 ? (1u << (n - 32)) - 1u : 0u;
            wait(kKVFull + k % kBufs, k / kBufs);  // (long since: what the unpacking warps wrote beside K and V is visible behind it)
#pragma unroll
            for (int c = 0; c < kG; ++c)
              if ((s_nan[k % kBufs][c][0] & v0) | (s_nan[k % kBufs][c][1] & v1)) poison |= 1u << c;
            __syncwarp();
          }
#pragma unroll
          for (int c = 0; c < 32; ++c) sr[0][c] = (v0 & (1u << c)) ? sr[0][c] : 0xff800000u;
          if (two) {
#pragma unroll
            for (int c = 0; c < 32; ++c) sr[1][c] = (v1 & (1u << c)) ? sr[1][c] : 0xff800000u;
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 32; c += 2) mx4[(c >> 1) & 3] = ptx::max3(mx4[(c >> 1) & 3], __uint_as_float(sr[0][c]), __uint_as_float(sr[0][c + 1]));
        if (two) {
#pragma unroll
          for (int c = 0; c < 32; c += 2) mx4[(c >> 1) & 3] = ptx::max3(mx4[(c >> 1) & 3], __uint_as_float(sr[1][c]), __uint_as_float(sr[1][c + 1]));
        }
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sl2;
        float m_new = fmaxf(m_run, mx);
        if (m_run != -INFINITY && m_new - m_run <= kLazy) m_new = m_run;
        const float ref = m_new == -INFINITY ? 0.f : m_new;
        const float corr = ptx::ex2(m_run - ref);
        const bool changed = m_new != m_run;
        m_run = m_new;
        const ptx::f32x2 sc2 = ptx::pack2(sl2, sl2), nr2 = ptx::pack2(-ref, -ref);
        ptx::f32x2 sum2[2] = {0ull, 0ull};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1 && !two) break;
          uint32_t parts[32];  // higher bits of 32 tokens, then what they leave
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float t0, t1;
            ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(sr[h][c]), __uint_as_float(sr[h][c + 1])), sc2, nr2), t0, t1);
            const float p0 = ptx::ex2(t0), p1 = ptx::ex2(t1);
            sum2[(c >> 1) & 1] = ptx::add2(sum2[(c >> 1) & 1], ptx::pack2(p0, p1));
            parts[c >> 1] = pack_bf16(p0, p1);
            parts[16 + (c >> 1)] = low_part(parts[c >> 1], p0, p1);
          }
          ptx::tmem_st32(tm_s + 32 * h, parts);
        }
        if (j > 0 && __any_sync(0xffffffffu, changed)) {  // (rare)
          wait(kODone + 2 * x + ((j - 1) & 1), (j - 1) >> 1);
          ptx::tc_fence_after_sync();
          __syncwarp();
#pragma unroll 1
          for (int ch = 0; ch < D / 32; ++ch) {
            uint32_t o[32];
            ptx::tmem_ld32(tm + kColO + (uint32_t)ch * 32, o);
            ptx::tmem_wait_ld(o);
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * corr);
            ptx::tmem_st32(tm + kColO + (uint32_t)ch * 32, o);
          }
        }
        float s0, s1, s2, s3;
        ptx::unpack2(sum2[0], s0, s1);
        ptx::unpack2(sum2[1], s2, s3);
        l_run = l_run * corr + ((s0 + s1) + (s2 + s3));
        ptx::tmem_wait_st();
        ptx::tc_fence_before_sync();
        __syncwarp();
        ptx::mbar_arrive_warp(bar(kPFull + 2 * x + (j & 1)));
      }
      if (!kLong || !s_more) break;
      meet();
      meet();
    }
    if (pages > 0) {
      wait(kODone + 2 * x + ((pages - 1) & 1), (pages - 1) >> 1);
      ptx::tc_fence_after_sync();
      __syncwarp();
    }
    // ---- the groups' parts of one tile: the second's through the place of K and V into the first's ----
    float4* const box = reinterpret_cast<float4*>(smem + SM::kKV);  // [D / 4][kTile]
    float4* const box_ml = box + D / 4 * kTile;                    // [kTile]: maximum, sum, groups with NaN
    float f0 = 1.f, f1 = 0.f;
    if (split) {
      asm volatile("bar.sync 2, 256;" ::: "memory");  // (every product has been made)
      if (x == 1) {
#pragma unroll 1
        for (int ch = 0; ch < D / 32; ++ch) {
          uint32_t o[32];
          if (pages > 0) {
            ptx::tmem_ld32(tm + kColO + (uint32_t)ch * 32, o);
            ptx::tmem_wait_ld(o);
          } else {
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = 0;
          }
#pragma unroll
          for (int c = 0; c < 32; c += 4)
            box[(ch * 8 + c / 4) * kTile + rr] =
                make_float4(__uint_as_float(o[c]), __uint_as_float(o[c + 1]), __uint_as_float(o[c + 2]), __uint_as_float(o[c + 3]));
        }
        box_ml[rr] = make_float4(m_run, l_run, __uint_as_float(poison), 0.f);
      }
      asm volatile("bar.sync 2, 256;" ::: "memory");
      if (x == 0) {
        const float4 other = box_ml[rr];
        const float top = fmaxf(m_run, other.x), ref = top == -INFINITY ? 0.f : top;
        f0 = ptx::ex2(m_run - ref);
        f1 = ptx::ex2(other.x - ref);
        m_run = top;
        l_run = l_run * f0 + other.y * f1;
        poison |= __float_as_uint(other.z);
      } else {  // a row that is not there
        r = row0 + tid;
        there = false;
        pages = 0;
      }
    }
    // ---- output: 32 columns at a time through the tile's place of Q, so that rows are written in pieces of 16 channels ----
    // Column 64 w + 8 g + 2 k + h of O is channel 32 (2 w + h) + 4 g + k: the order in which V's codes lie in a word.
    const int tok = r / G, hd = kvh * G + r % G;
    const int64_t row = ((int64_t)b * a.N + hd) * a.Lq + tok;
    const float inv = a.shares > 1 ? 1.f : l_run != 0.f ? 1.f / l_run : 0.f;  // (a sum that is NaN stays one)
    f0 *= inv;
    f1 *= inv;
    char* to = nullptr;
    if (tok < a.Lq) {
      if (a.shares == 1)
        to = reinterpret_cast<char*>(reinterpret_cast<__nv_bfloat16*>(a.o.ptr) + (int64_t)b * a.o.sb + (int64_t)hd * a.o.sh + (int64_t)tok * a.o.ss);
      else if (there && s_known > 0) to = reinterpret_cast<char*>(a.part_o + (row * a.shares + share) * D);
    }
    char* line_to[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      line_to[i] = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), 4 * i + (lane >> 3)));
    unsigned char* const stage = smem + x * SM::kQ + (warp & 3) * 4096;
#pragma unroll 1
    for (int ch = 0; ch < D / 32; ++ch) {
      float v[32];
      {
        uint32_t o[32];
        if (pages > 0) {
          ptx::tmem_ld32(tm + kColO + (uint32_t)ch * 32, o);
          ptx::tmem_wait_ld(o);
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(o[c]) * f0;
      }
      if (split && x == 0) {
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float4 w = box[(ch * 8 + c) * kTile + rr];
          v[4 * c] = fmaf(w.x, f1, v[4 * c]);
          v[4 * c + 1] = fmaf(w.y, f1, v[4 * c + 1]);
          v[4 * c + 2] = fmaf(w.z, f1, v[4 * c + 2]);
          v[4 * c + 3] = fmaf(w.w, f1, v[4 * c + 3]);
        }
      }
      const unsigned nan = poison >> (2 * (ch >> 1)) & 3;
      if (nan) {
#pragma unroll
        for (int c = 0; c < 32; ++c)
          if (nan >> (c & 1) & 1) v[c] = NAN;
      }
      if (!there || pages == 0) {
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = 0.f;
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {  // channels 16 (ch % 2) + 4 (c % 4) + 0..3 of group 2 (ch / 2) + c / 4
        const int k = 8 * (c & 3) + (c >> 2);
        *reinterpret_cast<float4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_float4(v[k], v[k + 2], v[k + 4], v[k + 6]);
      }
      __syncwarp();
      float4 piece[8];
      const int c = lane & 7, channel = 64 * (ch >> 1) + 32 * (c >> 2) + 16 * (ch & 1) + 4 * (c & 3);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int line = 4 * i + (lane >> 3);
        piece[i] = *reinterpret_cast<const float4*>(stage + line * 128 + ((c ^ (line & 7)) << 4));
      }
      if (a.shares > 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (line_to[i]) store4(reinterpret_cast<float*>(line_to[i]) + channel, piece[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (line_to[i]) store4(reinterpret_cast<__nv_bfloat16*>(line_to[i]) + channel, piece[i]);
      }
      __syncwarp();
    }
    if (tok < a.Lq) {
      if (!there) m_run = -INFINITY, l_run = 0.f;
      if (a.shares > 1) {
        if (there || sh.bad) a.part_ml[row * a.shares + share] = make_float2(m_run, l_run);
      } else if (a.lse) {
        a.lse[row] = l_run != 0.f ? (m_run + log2f(l_run)) * kLn2 : -INFINITY;
      }
    }
  } else if (warp < kMmaWarp) {
    // =============================== codes -> K and V ===========================================
    const int p = tid - 32 * kSoftWarps, t = p & 3, line = p >> 2;  // token pair `line`, and (eight lanes that write at once: other banks):
    const int key = (line & ~7) | (line & 1) << 2 | (line >> 1 & 3), flip = line & 1;  // keys `key`, `key` + 32; V's pieces 2 t + flip, then the other
    const unsigned char* const head = a.pages + (int64_t)kvh * L::kBytes;
    const Codes codes = a.codes;
    unsigned char* const cells = smem + SM::kCodes + p * SM::kCell;  // cell c of stage s: s kStage + c 128 kCell on
    unsigned char* const scale_cells = smem + SM::kCodes + 5 * 128 * SM::kCell + p * SM::kScales;
    auto request = [&](int k, int known) {
      if (k < known) {
        const int i = s_list[place(k)];
        const bool two = s_mask[2 * i + 1] != 0, pair = two || line < 16;
        const unsigned char* const page = head + (int64_t)s_page[i] * a.Nk * L::kBytes;
        const int stage = k % kAhead * SM::kStage;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (y == 0 || two) {
            cp_async<SM::kCell>(cells + stage + y * 128 * SM::kCell, page + L::k_word(key + 32 * y, 0, t));
            cp_async<SM::kScales>(scale_cells + stage + y * 128 * SM::kScales, page + L::k_scale(key + 32 * y, 0));
          }
          if (pair) cp_async<SM::kCell>(cells + stage + (2 + y) * 128 * SM::kCell, page + L::v_word(2 * line, 2 * t + (y ^ flip), 0));
        }
        if (pair) cp_async<SM::kCell>(cells + stage + 4 * 128 * SM::kCell, page + L::v_scale(2 * line, 0));
      }
      cp_async_commit();
    };
    int k = 0, page0 = sh.page0;
#pragma unroll 1
    for (;;) {
      const int known = s_known;
#pragma unroll 1
      for (int i = 0; i < kAhead - 1; ++i) request(k + i, known);
#pragma unroll 1
      for (; k < known; ++k) {
        const int buf = k % kBufs, i = s_list[place(k)], slot0 = (page0 + i) * kPage;
        const uint32_t in = s_mask[2 * i + (line >> 4)] >> (2 * line & 31);  // of this pair of tokens
        const bool late = slot0 + kPage - 1 > first_lim, two = s_mask[2 * i + 1] != 0, pair = two || line < 16;
        request(k + kAhead - 1, known);
        cp_async_wait<kAhead - 1>();  // this thread's cells of page k have landed
        uint32_t kw[2][kG], ks[2][kG / 2], vw[2][kG], vs[kG];
        {
          const int stage = k % kAhead * SM::kStage;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            load_words<D>(cells + stage + y * 128 * SM::kCell, kw[y]);
            load_words<D>(cells + stage + (2 + y) * 128 * SM::kCell, vw[y]);  // the even token's words, then the odd one's
            load_scales<D>(scale_cells + stage + y * 128 * SM::kScales, ks[y]);
          }
          load_words<D>(cells + stage + 4 * 128 * SM::kCell, vs);
        }
        if (k >= kBufs) wait(kKVEmpty + buf, k / kBufs - 1);
        unsigned char* const out_k = smem + SM::kKV + buf * 2 * SM::kHalf;
        unsigned char* const out_v = out_k + SM::kHalf;
        auto place = [&](int row, int unit) { return (unit >> 3) * SM::kChunk + row * 128 + (((unit & 7) ^ (row & 7)) << 4); };
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          if (y == 1 && !two) break;
#pragma unroll
          for (int j = 0; j < kG; ++j) {
            const Pairs x = pairs_of(codes, kw[y][j], __byte_perm(ks[y][j / 2], 0, j % 2 ? 0x3232 : 0x1010));
            *reinterpret_cast<uint4*>(out_k + place(key + 32 * y, 4 * j + t)) = make_uint4(x.x[0], x.x[1], x.x[2], x.x[3]);
          }
        }
        // values of tokens in no block are zeros (0 x NaN would reach every row); so are NaN that some rows see and others do not:
        // those rows are told
        const uint32_t keep = ((in & 1) ? 0xFFFFu : 0u) | ((in & 2) ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int j = 0; j < kG; ++j) vs[j] &= keep;
        if (late) {
          if (p < 2 * kG) s_nan[buf][p / 2][p % 2] = 0;
          unpackers_meet();
#pragma unroll
          for (int j = 0; j < kG; ++j) {
            const uint32_t is = __vcmpeq2(vs[j] & 0x7F807F80u, 0x7F807F80u);
            if (is && pair) atomicOr(&s_nan[buf][j][line >> 4], ((is & 1u) | ((is >> 31) << 1)) << (2 * line & 31));
            vs[j] &= ~is;
          }
        }
        if (pair) {
#pragma unroll
          for (int w = 0; w < kG / 2; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // the even and the odd token
              const uint32_t s2 = __byte_perm(vs[2 * w], vs[2 * w + 1], h ? 0x7632 : 0x5410), c2 = scale_offset(s2);
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const uint32_t x = vw[y][h * (kG / 2) + w];
                *reinterpret_cast<uint4*>(out_v + place(2 * line + h, 8 * w + 2 * t + (y ^ flip))) =
                    make_uint4(held(codes, x, s2, c2), held(codes, rotr(x, 4), s2, c2), held(codes, rotr(x, 8), s2, c2), held(codes, rotr(x, 12), s2, c2));
              }
            }
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        ptx::mbar_arrive_warp(bar(kKVFull + buf));
      }
      cp_async_wait<0>();
      if (!kLong || !s_more) break;
      meet();
      page0 += kAtOnce;
      find_pages(a, lists_of(a, b), s_prompt, page0, min(sh.page0 + sh.n - page0, kAtOnce), p, 32 * kUnpackWarps, s_mask, s_page);
      unpackers_meet();
      if (warp == kSoftWarps) make_list(page0, known);
      meet();
    }
  } else {
    // =============================== MMA ===========================================
    const uint32_t idesc_qk = ptx::idesc_bf16(kTile, kPage, 0, 0), idesc_half = ptx::idesc_bf16(kTile, kPage / 2, 0, 0), idesc_pv = ptx::idesc_bf16(kTile, D, 0, 1);
    const uint64_t q_desc = ptx::smem_desc_sw128(sbase, 16, 1024), k_desc = ptx::smem_desc_sw128(sbase + SM::kKV, 16, 1024);
    const uint64_t v_desc = ptx::smem_desc_sw128(sbase + SM::kKV + SM::kHalf, SM::kChunk, 1024);
    auto is_long = [&](int k) { return s_mask[2 * s_list[place(k)] + 1] != 0; };  // page k, beyond its first half
    // Page k for group x's tile: its j-th.
    auto issue_qk = [&](int k, int x, int j) {
      const int buf = k % kBufs;
      const uint32_t idesc = is_long(k) ? idesc_qk : idesc_half;
      wait(kKVFull + buf, k / kBufs);
      ptx::tc_fence_after_sync();
      __syncwarp();
      if (ptx::elect_one()) {
        const uint32_t d = tmem + (uint32_t)x * kTileCols + (uint32_t)(j & 1) * 64, q = (uint32_t)q_desc + (split ? 0u : (uint32_t)x * (SM::kQ >> 4));
        const uint32_t key = (uint32_t)k_desc + (uint32_t)buf * (2 * SM::kHalf >> 4);
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
          ptx::mma_ss_lohi(d, q + (s >> 2) * (SM::kQChunk >> 4) + (s & 3) * 2, (uint32_t)(q_desc >> 32), key + (s >> 2) * (SM::kChunk >> 4) + (s & 3) * 2,
                           (uint32_t)(k_desc >> 32), idesc, s > 0);
        ptx::mma_commit(bar(kSFull + 2 * x + (j & 1)));
      }
      __syncwarp();
    };
    auto issue_pv = [&](int k, int x, int j, bool last) {
      const int buf = k % kBufs;
      const bool two = is_long(k);
      wait(kPFull + 2 * x + (j & 1), j >> 1);
      ptx::tc_fence_after_sync();
      __syncwarp();
      if (ptx::elect_one()) {
        const uint32_t s = tmem + (uint32_t)x * kTileCols + (uint32_t)(j & 1) * 64, d = tmem + (uint32_t)x * kTileCols + kColO;
        const uint32_t v = (uint32_t)v_desc + (uint32_t)buf * (2 * SM::kHalf >> 4);
#pragma unroll
        for (int ks = 0; ks < kPage / 16; ++ks) {
          if (ks == kPage / 32 && !two) break;
          const uint32_t p = s + (ks >> 1) * 32 + (ks & 1) * 8;
          ptx::mma_ts_lohi(d, p, v + ks * (16 * 128 >> 4), (uint32_t)(v_desc >> 32), idesc_pv, j > 0 || ks > 0);
          ptx::mma_ts_lohi(d, p + 16, v + ks * (16 * 128 >> 4), (uint32_t)(v_desc >> 32), idesc_pv, 1u);
        }
        ptx::mma_commit(bar(kODone + 2 * x + (j & 1)));
        if (last) ptx::mma_commit(bar(kKVEmpty + buf));
      }
      __syncwarp();
    };
    int k = 0;
#pragma unroll 1
    for (;;) {
      const int known = s_known;
      if (split) {
#pragma unroll 1
        for (int n = k; n < min(known, k + 2); ++n) issue_qk(n, n & 1, n >> 1);
#pragma unroll 1
        for (; k < known; ++k) {
          issue_pv(k, k & 1, k >> 1, true);
          if (k + 2 < known) issue_qk(k + 2, k & 1, (k >> 1) + 1);
        }
      } else {
        if (k < known)
          for (int x = 0; x < 2; ++x) issue_qk(k, x, k);
#pragma unroll 1
        for (; k < known; ++k) {
          if (k + 1 < known)
            for (int x = 0; x < 2; ++x) issue_qk(k + 1, x, k + 1);
          for (int x = 0; x < 2; ++x) issue_pv(k, x, k, x == 1);
        }
      }
      if (!kLong || !s_more) break;
      meet();
      meet();
    }
  }
  ptx::tc_fence_before_sync();
  ptx::end_of_waits(waits, [](int) { return kStatusCacheWait; }, a.status);
  if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, kTmemCols);
}

}  // namespace

int cache_attn_tc_launch(const cache::CacheAttnArgs& a, int D, cudaStream_t st) {
  const int64_t rows = (int64_t)a.Lq * (a.N / a.Nk), z = (rows + 2 * kTile - 1) / (2 * kTile);
  const dim3 grid(a.shares, a.B * a.Nk, (unsigned)z);
  auto run = [&](auto kern, int bytes, std::atomic<bool>* configured) -> int {
    int dev = 0;
    BRK_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
      BRK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    return launch_dependent(kern, grid, dim3(kThreads), bytes, st, a);
  };
  static std::atomic<bool> done[4][64] = {};
  constexpr int k128 = Smem<128>::kBytes + 1024, k64 = Smem<64>::kBytes + 1024;
  if ((a.P + a.shares - 1) / a.shares > kAtOnce)
    return D == 128 ? run(cache_attn_tc_kernel<128, true>, k128, done[0]) : run(cache_attn_tc_kernel<64, true>, k64, done[1]);
  return D == 128 ? run(cache_attn_tc_kernel<128, false>, k128, done[2]) : run(cache_attn_tc_kernel<64, false>, k64, done[3]);
}

}  // namespace brk
