// Layout of the 4-bit cache and the pieces that its kernels share.
//
// A page holds 64 tokens of one KV head: K codes, K scales, V codes, V scales, one behind the other.  Per (token, 32 channels)
// there is a scale s with 5 significant bits and 8 exponent bits (stored as bf16) and a code u = n + 8 per channel, n in -7..7;
// the value is n s.
//
// Both products take the codes as they are, without rounding:
//
// V: 3 bits of n times 5 bits of s fit the 8 significant bits of bf16, and one instruction per two values makes them: with u in bits
// 3..6 of a bf16 whose exponent is that of 16, the number is 16 + u = 24 + n, and fma(24 + n, s, -24 s) = n s is exact (24 s has 7
// significant bits).
//
// K: the scale of a group can wait for the sum over its channels, so the codes go in as numbers: the low 8 bits of a bf16, its
// mantissa and its lowest exponent bit, are one even grid (subnormals and the binade above them), so a code in bits 0..3 is u 2^-133 and
// one in bits 4..7 16 u 2^-133 by a mask alone.  The query is scaled by a power of two (exact) that brings its largest magnitude to
// 2^120, and by 1/16 where it meets the latter; -8 sum(q) s, summed over the groups, is one more product, of the scales.
// The order inside a row follows the MMA fragments, lane = 4 g + t, so that every lane's codes are one load:
//   K  row r (D/2 bytes): word t (D/32) + j holds channels 32 j + 8 t + 0..7.  Lane (g, t) reads the D/32 words of key g from
//      its quarter on: A (16 keys x the channels of group j), in whatever order Q has them too.
//   V  tokens 2p, 2p + 1 (D bytes): piece g (D/8 bytes) holds channels 32 j + 4 g + 0..3 of both tokens, first all of 2p's.
//      Lane (g, t) reads the piece g of pair t: A (16 channels x 16 keys), two keys of a register side by side.  Words are
//      stored rotated by 3 bits to the left: whole bytes and shifts by 4 bring any code to bits 3..6.
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

// For V: bits 3..6 of both halves of a word, and 16.0 in both.  An argument of the kernels: of constants that it knows the assembler makes
// two instructions for every (x & mask) | base, since only one operand can be a constant.
struct Codes {
  uint32_t mask = 0x00780078u, base = 0x41804180u;
};

__device__ __forceinline__ uint32_t rotr(uint32_t x, int n) { return __funnelshift_r(x, x, n); }
__device__ __forceinline__ uint32_t rotl(uint32_t x, int n) { return __funnelshift_l(x, x, n); }

__device__ __forceinline__ uint32_t fma_bf2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t mul_bf2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t add_bf2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// -24 s, for two scales
__device__ __forceinline__ uint32_t scale_offset(uint32_t s2) { return mul_bf2(s2, 0xC1C0C1C0u); }
// two codes in bits 3..6 and 19..22 of x (others are ignored) -> their values
__device__ __forceinline__ uint32_t held(const Codes& k, uint32_t x, uint32_t s2, uint32_t c2) {
  return fma_bf2((x & k.mask) | k.base, s2, c2);
}

// a word of 8 codes -> their values, k and k + 4 in one register
struct Pairs {
  uint32_t x[4];
};
__device__ __forceinline__ Pairs pairs_of(const Codes& codes, uint32_t w, uint32_t s2) {
  const uint32_t c2 = scale_offset(s2);
  Pairs p;
#pragma unroll
  for (int k = 0; k < 4; ++k) p.x[k] = held(codes, rotl(w, (35 - 4 * k) % 32), s2, c2);
  return p;
}
__device__ __forceinline__ uint2 low_values(const Pairs& p) { return make_uint2(__byte_perm(p.x[0], p.x[1], 0x5410), __byte_perm(p.x[2], p.x[3], 0x5410)); }
__device__ __forceinline__ uint2 high_values(const Pairs& p) { return make_uint2(__byte_perm(p.x[0], p.x[1], 0x7632), __byte_perm(p.x[2], p.x[3], 0x7632)); }

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

template <int D>
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&w)[D / 32]) {
  if constexpr (D == 128) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
  else *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
}
template <int D>
__device__ __forceinline__ void load_scales(const unsigned char* p, uint32_t (&w)[D / 64]) {
  if constexpr (D == 128) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
  else w[0] = *reinterpret_cast<const uint32_t*>(p);
}

// The rows of a warp as the 8-column operand: 8 kTiles columns of queries, one row each, and their products with pages of keys.
// A bf16 query is one bf16 number, an fp32 one three.  Logits are to be multiplied by `unit` (by tile and by which of the two
// columns of a C fragment): each row's power of two.
template <typename T, int D, int kTiles>
struct QueryRows {
  using L = Layout<D>;
  static constexpr int kPieces = sizeof(T) == 4 ? 3 : 1;
  // fp32: -8 is added to the codes instead (-8 2^-133 and -128 2^-133): of sums of n q, not of u q, fewer bits cancel.  (Output's error
  // against 64 bits, 2 prompts of 100 documents, head_dim 64: 1.1e-6 with the codes as they are and one sum per group,
  // 0.6e-6 so and with sums of 16 channels; plain fp32 0.5e-6.)
  static constexpr bool kSigned = sizeof(T) == 4;
  uint32_t q[kTiles][kPieces][L::kGroups][2][2];  // [group][step][register]: channels 8 t + 2 step + {0, 4}, {1, 5}
  uint32_t shift[kTiles][2];                      // B of the product of the scales: -8 2^-133 sum(q) of the groups, in three bf16 numbers
  float unit[kTiles][2];

  // this lane's channels of the queries as they are in memory, so that they can be on their way while something else is done
  struct Raw {
    uint4 w[kTiles][L::kGroups][sizeof(T) / 2];
  };
  // row(c): column c's query, null for none
  template <typename F>
  static __device__ __forceinline__ void fetch(F row, int g, int t, Raw& raw) {
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      const T* const p = row(8 * n + g);
#pragma unroll
      for (int j = 0; j < L::kGroups; ++j)
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
          raw.w[n][j][i] = p ? *(reinterpret_cast<const uint4*>(p + 32 * j + 8 * t) + i) : make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void make(const Raw& raw, int g, int t) {
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      // the bits of the row's largest magnitude (NaN is above infinity)
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < L::kGroups; ++j)
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
          const uint4 w = raw.w[n][j][i];
          if constexpr (sizeof(T) == 2) {
            const uint32_t k = 0x7FFF7FFFu;
            top = __vmaxu2(top, __vmaxu2(__vmaxu2(w.x & k, w.y & k), __vmaxu2(w.z & k, w.w & k)));
          } else {
            const uint32_t k = 0x7FFFFFFFu;
            top = max(top, max(max(w.x & k, w.y & k), max(w.z & k, w.w & k)));
          }
        }
      if constexpr (sizeof(T) == 2) top = max(top & 0xFFFF0000u, top << 16);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^up = 2^120 / 2^(exponent of top); in two factors, since it can be 2^246
      const bool finite = top < 0x7F800000u;
      const int up = 120 + 127 - (int)max(top >> 23, 1u);
      const uint32_t up0 = (uint32_t)(up / 2 + 127) << 23, up1 = (uint32_t)(up - up / 2 + 127) << 23;  // (as numbers)
      float total[L::kGroups];
#pragma unroll
      for (int j = 0; j < L::kGroups; ++j) {
        if constexpr (sizeof(T) == 2) {
          // powers of two leave bf16 as it is: packed
          const uint32_t u0 = up0 | up0 >> 16, u1 = up1 | up1 >> 16, none = finite ? ~0u : 0u;
          const uint4 w = raw.w[n][j][0];
          const uint32_t x[4] = {mul_bf2(mul_bf2(w.x & none, u0), u1), mul_bf2(mul_bf2(w.y & none, u0), u1),
                                 mul_bf2(mul_bf2(w.z & none, u0), u1), mul_bf2(mul_bf2(w.w & none, u0), u1)};
          total[j] = ((bf_lo(x[0]) + bf_hi(x[0])) + (bf_lo(x[1]) + bf_hi(x[1]))) + ((bf_lo(x[2]) + bf_hi(x[2])) + (bf_lo(x[3]) + bf_hi(x[3])));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            q[n][0][j][h][0] = __byte_perm(x[h], x[h + 2], 0x5410);
            q[n][0][j][h][1] = mul_bf2(__byte_perm(x[h], x[h + 2], 0x7632), 0x3D803D80u);  // 1/16
          }
        } else {
          float x[8];
          load8(reinterpret_cast<const float*>(raw.w[n][j]), x);
          total[j] = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            x[k] = finite ? x[k] * __uint_as_float(up0) * __uint_as_float(up1) : 0.f;
            total[j] += x[k];
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t piece[kPieces];
            const float f = k % 2 ? 0.0625f : 1.f;
            split2<kPieces>(x[k] * f, x[k + 4] * f, piece);
#pragma unroll
            for (int i = 0; i < kPieces; ++i) q[n][i][j][k / 2][k % 2] = piece[i];
          }
        }
        total[j] += __shfl_xor_sync(0xffffffffu, total[j], 1);
        total[j] += __shfl_xor_sync(0xffffffffu, total[j], 2);
        total[j] *= -0x1p-126f * 0x1p-4f;  // (about 2^-5)
      }
      // The scales stand side by side in A as they do in memory, the groups' four times (D 128) or eight times over.
      uint32_t w[3][L::kGroups / 2];
#pragma unroll
      for (int j = 0; j < L::kGroups; j += 2) {
        uint32_t piece[3];
        split2<3>(total[j], total[j + 1], piece);
#pragma unroll
        for (int i = 0; i < 3; ++i) w[i][j / 2] = piece[i];
      }
      if constexpr (D == 128) {
        shift[n][0] = t == 0 ? w[0][0] : t == 1 ? w[0][1] : t == 2 ? w[1][0] : w[1][1];
        shift[n][1] = t == 0 ? w[2][0] : t == 1 ? w[2][1] : 0u;
      } else {
        shift[n][0] = t == 0 ? w[0][0] : t == 1 ? w[1][0] : t == 2 ? w[2][0] : 0u;
        shift[n][1] = 0u;
      }
      // 2^(133 - up), up >= -7: a row with NaN or an infinity has a unit of NaN, one with a magnitude from 2^115 on of infinity (its logits
      // are infinities or NaN)
      const float down = !finite ? NAN : 133 - up > 127 ? INFINITY : up > 133 + 126 ? 0.f : __uint_as_float((uint32_t)(133 - up + 127) << 23);
#pragma unroll
      for (int y = 0; y < 2; ++y) unit[n][y] = __shfl_sync(0xffffffffu, down, 4 * (2 * t + y));
    }
  }
  // What logits of tile n's columns x are multiplied by to be exponents of 2.  Never 0 (a row of zeros has the smallest unit, 2^-113, and a
  // scale can be smaller still): the running maximum begins at -infinity.
  __device__ __forceinline__ float exponent_scale(float scale, int n, int x) const {
    const float f = scale * 1.4426950408889634f * unit[n][x];
    return f == 0.f ? 0x1p-149f : f;
  }
  // s[n][i]: the C fragment of keys 16 i .. 16 i + 15 of the page and the columns of tile n
  __device__ __forceinline__ void logits(const unsigned char* page, int g, int t, float (&s)[kTiles][4][4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t wa[L::kGroups], wb[L::kGroups], sa[L::kGroups / 2], sb[L::kGroups / 2];
      load_words<D>(page + L::k_word(16 * i + g, 0, t), wa);
      load_words<D>(page + L::k_word(16 * i + 8 + g, 0, t), wb);
      load_scales<D>(page + L::k_scale(16 * i + g, 0), sa);
      load_scales<D>(page + L::k_scale(16 * i + 8 + g, 0), sb);
      if constexpr (kSigned) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][i][x] = 0.f;
      } else {
        const uint32_t a = D == 128 && t % 2 ? sa[L::kGroups / 2 - 1] : sa[0], b = D == 128 && t % 2 ? sb[L::kGroups / 2 - 1] : sb[0];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][i][x] = 0.f;
          mma(s[n][i], a, b, a, b, shift[n][0], shift[n][1]);
        }
      }
#pragma unroll
      for (int j = 0; j < L::kGroups; ++j) {
        const float fa = j % 2 ? bf_hi(sa[j / 2]) : bf_lo(sa[j / 2]), fb = j % 2 ? bf_hi(sb[j / 2]) : bf_lo(sb[j / 2]);
        const uint32_t a8 = wa[j] >> 8, b8 = wb[j] >> 8;
        uint32_t a[4] = {wa[j] & 0x000F000Fu, wa[j] & 0x00F000F0u, a8 & 0x000F000Fu, a8 & 0x00F000F0u};  // codes k and k + 4
        uint32_t b[4] = {wb[j] & 0x000F000Fu, wb[j] & 0x00F000F0u, b8 & 0x000F000Fu, b8 & 0x00F000F0u};
        if constexpr (kSigned) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            a[k] = add_bf2(a[k], k % 2 ? 0x80808080u : 0x80088008u);
            b[k] = add_bf2(b[k], k % 2 ? 0x80808080u : 0x80088008u);
          }
        }
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          // The tensor cores cut a sum off where it would have to be rounded: in fp32 the products with the first pieces, 16 channels each, are
          // sums of their own, added in 32 bits.
          float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = kPieces - 1; p >= 0; --p)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if constexpr (kPieces == 1) {
                mma(x, a[2 * h], b[2 * h], a[2 * h + 1], b[2 * h + 1], q[n][p][j][h][0], q[n][p][j][h][1]);
              } else {
                float y[4] = {0.f, 0.f, 0.f, 0.f};
                float (&sum)[4] = p > 0 ? x : y;
                mma(sum, a[2 * h], b[2 * h], a[2 * h + 1], b[2 * h + 1], q[n][p][j][h][0], q[n][p][j][h][1]);
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  if (p == 0) x[z] += y[z];
              }
            }
#pragma unroll
          for (int z = 0; z < 4; ++z) s[n][i][z] = fmaf(x[z], z < 2 ? fa : fb, s[n][i][z]);
        }
      }
    }
  }
};

// One prompt's block spans, read by all threads of a CTA: `bad` if a block lies outside [0, slots), has a negative length or
// begins before the end of the one in front of it.
__device__ __forceinline__ bool span_is_bad(const int32_t* start, const int32_t* len, int m, int64_t slots) {
  const int64_t s = start[m], n = len[m];
  return s < 0 || n < 0 || s + n > slots || (m > 0 && s < (int64_t)start[m - 1] + len[m - 1]);
}

}  // namespace cache
}  // namespace brk
