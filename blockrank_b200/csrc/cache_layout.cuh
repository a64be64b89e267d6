// Layout of the 4-bit cache and the pieces that its kernels share.
//
// A page holds 64 tokens of one KV head: K codes, K scales, V codes, V scales, one behind the other.  Per (token, 32 channels)
// there is a scale s with 5 significant bits and 8 exponent bits (stored as bf16) and a code u = n + 8 per channel, n in -7..7;
// the value is n s.
//
// 3 bits of n times 5 bits of s fit the 8 significant bits of bf16, so the tensor cores get the held values themselves, unrounded,
// and one instruction per two values makes them: with u in bits 3..6 of a bf16 whose exponent is that of 16, the number is
// 16 + u = 24 + n, and fma(24 + n, s, -24 s) = n s is exact (24 s has 7 significant bits).  Hence every 32-bit word of codes is
// stored rotated by 3 bits to the left: a shift by a multiple of 4 brings any code there.  (A scale with all 8 bits of bf16
// would have to be applied behind the product: for V once per group of 32 channels to each probability and both parts that
// it is split into, for K to every accumulator; counted from the source 351 instructions per 16 keys instead of 287.)
//
// The order inside a row follows the fragments of mma.m16n8k16, lane = 4 g + t, so that every lane's codes are one load:
//   K  row r (D/2 bytes): word t (D/32) + j holds channels 32 j + 8 t + 0..7.  Lane (g, t) reads the D/32 words of key g from
//      its quarter on: A (16 keys x 16 channels), where a step's channels are two of each t's, in whatever order Q has too.
//   V  tokens 2p, 2p + 1 (D bytes): piece g (D/8 bytes) holds channels 32 j + 4 g + 0..3 of both tokens, first all of 2p's.
//      Lane (g, t) reads the piece g of pair t: A (16 channels x 16 keys), two keys of a register side by side.
//   scales: K [64][D/32]; V [32 pairs][D/32][2 tokens].
#pragma once
#include "brk_common.cuh"
#include "mma_bf16.cuh"

namespace brk {
namespace cache {

constexpr int kPage = BRK_CACHE_PAGE;  // tokens
constexpr int kGroup = 32;             // channels that share a scale

template <int D>
struct Layout {
  static constexpr int kGroups = D / kGroup;
  static constexpr int kCodes = kPage * D / 2;            // bytes of a page's K (or V) codes
  static constexpr int kScales = kPage * kGroups * 2;     // ... scales
  static constexpr int kHalf = kCodes + kScales;          // K part, then V part
  static constexpr int kBytes = 2 * kHalf;
  // byte offsets inside a page
  static __host__ __device__ constexpr int k_word(int tok, int j, int t) { return tok * (D / 2) + (t * kGroups + j) * 4; }
  static __host__ __device__ constexpr int k_scale(int tok, int j) { return kCodes + (tok * kGroups + j) * 2; }
  // the word with the channels 4 g + 0..3 of groups 2 w (low half) and 2 w + 1
  static __host__ __device__ constexpr int v_word(int tok, int g, int w) {
    return kHalf + (tok >> 1) * D + g * (D / 8) + (tok & 1) * (D / 16) + w * 4;
  }
  static __host__ __device__ constexpr int v_scale(int tok, int j) { return kHalf + kCodes + ((tok >> 1) * kGroups + j) * 4 + (tok & 1) * 2; }
};
inline size_t head_page_bytes(int D) { return D == 128 ? Layout<128>::kBytes : Layout<64>::kBytes; }

constexpr uint32_t kCodeMask = 0x00780078u, kCodeBase = 0x41804180u;  // bits 3..6 of both halves; 16.0 in both

__device__ __forceinline__ uint32_t rotr(uint32_t x, int n) { return __funnelshift_r(x, x, n); }
__device__ __forceinline__ uint32_t rotl(uint32_t x, int n) { return __funnelshift_l(x, x, n); }

__device__ __forceinline__ uint32_t fma_bf2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// -24 s, for two scales
__device__ __forceinline__ uint32_t scale_offset(uint32_t s2) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(s2), "r"(0xC1C0C1C0u));
  return d;
}
// two codes in bits 3..6 and 19..22 of x (others are ignored) -> their values
__device__ __forceinline__ uint32_t held(uint32_t x, uint32_t s2, uint32_t c2) { return fma_bf2((x & kCodeMask) | kCodeBase, s2, c2); }

// C (16 x 8) += A (16 x 16) B (16 x 8)
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 matrix of 16-bit values, two of row lane / 4 in each lane -> its transpose
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
__device__ __forceinline__ float bf_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float bf_hi(uint32_t x) { return __uint_as_float(x & 0xFFFF0000u); }

// x = sum of kPieces bf16 numbers, each the rest behind the ones before it: 8, 16 or all 24 bits of x
template <int kPieces>
__device__ __forceinline__ void split2(float x0, float x1, uint32_t (&piece)[kPieces]) {
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    piece[i] = pack_bf16(x0, x1);
    if (i + 1 < kPieces) {
      x0 -= bf_lo(piece[i]);
      x1 -= bf_hi(piece[i]);
    }
  }
}

// The K part of a page (in shared memory) times kTiles x 8 query rows: s[n][i] is the C fragment of keys 16 i .. 16 i + 15 and
// rows 8 n .. 8 n + 7.  q[n][piece][j][h]: B fragment of group j's step h, channels 32 j + 8 t + 2 h + {0, 4} and {1, 5}.
template <int D, int kTiles, int kPieces>
__device__ __forceinline__ void page_logits(const unsigned char* page, const uint32_t (&q)[kTiles][kPieces][D / 32][2][2], int g, int t,
                                            float (&s)[kTiles][4][4]) {
  using L = Layout<D>;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t wa[L::kGroups], wb[L::kGroups], sa[L::kGroups / 2], sb[L::kGroups / 2];
    const unsigned char *ka = page + L::k_word(16 * i + g, 0, t), *kb = page + L::k_word(16 * i + 8 + g, 0, t);
    const unsigned char *ca = page + L::k_scale(16 * i + g, 0), *cb = page + L::k_scale(16 * i + 8 + g, 0);
    if constexpr (D == 128) {
      *reinterpret_cast<uint4*>(wa) = *reinterpret_cast<const uint4*>(ka);
      *reinterpret_cast<uint4*>(wb) = *reinterpret_cast<const uint4*>(kb);
      *reinterpret_cast<uint2*>(sa) = *reinterpret_cast<const uint2*>(ca);
      *reinterpret_cast<uint2*>(sb) = *reinterpret_cast<const uint2*>(cb);
    } else {
      *reinterpret_cast<uint2*>(wa) = *reinterpret_cast<const uint2*>(ka);
      *reinterpret_cast<uint2*>(wb) = *reinterpret_cast<const uint2*>(kb);
      sa[0] = *reinterpret_cast<const uint32_t*>(ca);
      sb[0] = *reinterpret_cast<const uint32_t*>(cb);
    }
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[n][i][x] = 0.f;
#pragma unroll
    for (int j = 0; j < L::kGroups; ++j) {
      const uint32_t s2a = __byte_perm(sa[j / 2], 0, j % 2 ? 0x3232 : 0x1010), s2b = __byte_perm(sb[j / 2], 0, j % 2 ? 0x3232 : 0x1010);
      const uint32_t c2a = scale_offset(s2a), c2b = scale_offset(s2b);
      uint32_t a[4], b[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        a[k] = held(rotr(wa[j], 4 * k), s2a, c2a);
        b[k] = held(rotr(wb[j], 4 * k), s2b, c2b);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int p = 0; p < kPieces; ++p) mma(s[n][i], a[2 * h], b[2 * h], a[2 * h + 1], b[2 * h + 1], q[n][p][j][h][0], q[n][p][j][h][1]);
    }
  }
}

// The B fragments of one query row for page_logits: this lane's channels 32 j + 8 t + 0..7 of the row at `p` (null: zeros).
template <int D, int kPieces>
__device__ __forceinline__ void load_query(const __nv_bfloat16* p, int t, uint32_t (&q)[kPieces][D / 32][2][2]) {
  static_assert(kPieces == 1, "bf16 needs no splitting");
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const uint4 w = p ? *reinterpret_cast<const uint4*>(p + 32 * j + 8 * t) : make_uint4(0, 0, 0, 0);
    q[0][j][0][0] = __byte_perm(w.x, w.z, 0x5410);
    q[0][j][0][1] = __byte_perm(w.x, w.z, 0x7632);
    q[0][j][1][0] = __byte_perm(w.y, w.w, 0x5410);
    q[0][j][1][1] = __byte_perm(w.y, w.w, 0x7632);
  }
}
template <int D, int kPieces>
__device__ __forceinline__ void load_query(const float* p, int t, uint32_t (&q)[kPieces][D / 32][2][2]) {
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    float x[8] = {};
    if (p) load8(p + 32 * j + 8 * t, x);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t piece[kPieces];
      split2<kPieces>(x[k], x[k + 4], piece);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) q[i][j][k / 2][k % 2] = piece[i];
    }
  }
}

// One prompt's block spans, read by all threads of a CTA: `bad` if a block lies outside [0, slots), has a negative length or
// begins before the end of the one in front of it.
__device__ __forceinline__ bool span_is_bad(const int32_t* start, const int32_t* len, int m, int64_t slots) {
  const int64_t s = start[m], n = len[m];
  return s < 0 || n < 0 || s + n > slots || (m > 0 && s < (int64_t)start[m - 1] + len[m - 1]);
}

}  // namespace cache
}  // namespace brk
