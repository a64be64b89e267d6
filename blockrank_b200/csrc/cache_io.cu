// The 4-bit cache: quantising keys and values as they are written, and reading them back.
//
// s = max|x| / 7 of a group of 32 channels, rounded to 5 significant bits (nearest, ties to even; never to a finer quantum than
// 2^-130; at most 1.9375 * 2^122), n = round(x / s) (ties to even) within -7..7.  Rounding s to the nearest never cuts the
// largest value off: 7 / (1 - 2^-5) < 7.5.
// Both decisions are those of exact arithmetic.  A border of n is (k + 1/2) s, 4 bits times 5; of s, a 6-bit number times 7:
// representable, so a 32-bit x is either equal to it or off by more than half a last place of the quotient, and a correctly
// rounded quotient lies on the border only if x does.  (Of a quotient that is a normal number; for others see group_scale().)  Where
// that costs too much, see quantise().
#include <algorithm>

#include "cache_layout.cuh"
#include "tc_ptx.cuh"

namespace brk {
namespace {

using namespace cache;

struct IoArgs {
  unsigned char* pages;
  View k, v;
  const int32_t* slots;
  int32_t* owner;  // where owner_place says: the last token of the call that names the slot; null: looked up in `slots`
  int32_t* key;    // a table by hash: the slot that a place is for, -1 for none; null: a place per slot of the pool
  int hash_shift;  // 32 - log2 of the table's places
  int32_t* status;
  int64_t n_slots;
  int tokens;  // B S
  int S, Nk;
  int tile;           // tokens of a CTA
  uint32_t per_head;  // 2^32 / Nk, rounded up (a row's number times it has its token in the high word: rows of a CTA times Nk < 2^32)
  Codes codes;
};

constexpr float kLargestScale = 1.9375f * 5316911983139663491615228241121378304.f;  // 2^122

__device__ __forceinline__ float reciprocal(float x) {  // 1 ulp
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// kN (8 or 4) channels of a lane as they are in memory
template <typename T, int kN>
struct Raw {
  static constexpr int kWords = kN * (int)sizeof(T) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void fetch(const T* p, bool there) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
    if (!there) return;
    if constexpr (kWords == 2) {
      const uint2 x = __ldcs(reinterpret_cast<const uint2*>(p));
      w[0] = x.x; w[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 x = __ldcs(reinterpret_cast<const uint4*>(p) + i / 4);
        w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
      }
    }
  }
  // the largest magnitude's bits (of its type): NaN is above infinity
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
      return max(m >> 16, m & 0xFFFFu);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
      return m;
    }
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return i % 2 ? bf_hi(w[i / 2]) : bf_lo(w[i / 2]);
  }
};

// The largest magnitudes of kGroups groups over kLanes (4 or 8) neighbouring lanes.
template <typename T, int kGroups, int kLanes>
__device__ __forceinline__ void reduce_largest(uint32_t (&m)[kGroups]) {
  if constexpr (sizeof(T) == 2) {  // two to a register
#pragma unroll
    for (int j = 0; j < kGroups; j += 2) {
      uint32_t x = m[j] | (m[j + 1] << 16);
#pragma unroll
      for (int off = 1; off < kLanes; off <<= 1) x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, off));
      m[j] = x & 0xFFFFu;
      m[j + 1] = x >> 16;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kGroups; ++j)
#pragma unroll
      for (int off = 1; off < kLanes; off <<= 1) m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], off));
  }
}

// The scale of a group whose largest magnitude has these bits, NaN where it holds NaN or an infinity.
// fp32 below 7 * 2^-126, where amax / 7 is subnormal and would be rounded before it is brought to the grid of 2^-130: the quotient is
// taken 2^32 times as large, and a sum with 1.5 * 2^-75, whose last place is 2^-98, rounds it once.
template <typename T>
__device__ __forceinline__ float group_scale(uint32_t top) {
  constexpr bool kBf16 = sizeof(T) == 2;
  if (kBf16) top <<= 16;
  const float amax = __uint_as_float(top);
  const bool fine = !kBf16 && amax < 0x1.cp-124f;
  uint32_t b = __float_as_uint(kBf16 ? amax * 0x1.24924ap-3f : __fdiv_rn(fine ? amax * 0x1p32f : amax, 7.f));
  if (kBf16) b = (b + 0x200u) & ~0x3FFu;
  float s = fminf(__uint_as_float((b + 0x3FFFFu + ((b >> 19) & 1u)) & ~0x7FFFFu), kLargestScale);
  if (fine) s = __fadd_rn(__fadd_rn(__uint_as_float(b), 0x1.8p-75f), -0x1.8p-75f) * 0x1p-32f;
  return top < 0x7F800000u ? s : NAN;
}

// kN values over a scale, as codes, value i in bits 4 i .. 4 i + 3; r: the reciprocal of the scale, 0 for a scale that is 0 or NaN.
//
// bf16: quotients by reciprocals (2^-22 of them off at most), rounded to 2^-13 of their unit first.  amax / 7 is on a border of s, and
// x / s on one of n, or 2^-9 of it away (8 bits against 9 of 7 times a border, of (k + 1/2) s), so the first rounding leaves
// it on the border or on its side.
// fp32: s by a division; `divide` is set where a quotient is within 2^-18 of a border.
template <typename T, int kN>
__device__ __forceinline__ uint32_t quantise(const Raw<T, kN>& x, float r, bool& divide) {
  // a sum with 1.5 * 2^23 + 8 has the rounded number + 8 in its low bits, on top of 0x4B400000
  constexpr float kInt = 12582920.f, kFine = 1536.f;
  constexpr uint32_t kOnTop = 0x4B400000u * (kN == 8 ? 0x11111111u : 0x1111u);
  uint32_t w = 0;
#pragma unroll
  for (int i = kN - 1; i >= 0; --i) {
    float n;
    if (sizeof(T) == 2) {
      n = __fadd_rn(__fmaf_rn(x.value(i), r, kFine), kInt - kFine);  // 1536 + a multiple of 2^-13, then a whole number
    } else {
      n = __fmaf_rn(x.value(i), r, kInt);
      divide |= fabsf(__fmaf_rn(x.value(i), r, -__fadd_rn(n, -kInt))) > 0.5f - 0x1p-18f;
    }
    w = w * 16 + __float_as_uint(n);
  }
  return w - kOnTop;
}
// The same by divisions, for any scale.
template <typename T, int kN>
__device__ __noinline__ uint32_t quantise_exactly(const Raw<T, kN> x, float s) {
  uint32_t w = 0;
#pragma unroll
  for (int i = kN - 1; i >= 0; --i) {
    const float n = s > 0.f ? rintf(__fdiv_rn(x.value(i), s)) : 0.f;
    w = w * 16 + (uint32_t)((int)fminf(fmaxf(n, -7.f), 7.f) + 8);
  }
  return w;
}

constexpr int kIoThreads = 256;
constexpr int kTile = 32;  // tokens of a CTA, at most
// Calls with at most this many tokens look for a later token with the same slot in the list itself; others go through `owner`, two
// kernels more.  (8 heads of 128: 32 tokens 2.9 us, with `owner` 4.3; 1024 4.3 and 5.4; 2048 6.6 and 6.1, but 4 us less from the host;
// 4096 14.5 and 8.3.)
constexpr int kScan = 2048;

// Places of a table by hash for so many tokens: a power of two, at most half of them taken.  It takes longer (16,384 tokens 32 us, with a
// place per slot of the pool 23.5; 78,720 91 and 83), so it is used for pools of more than 2^24 slots (64 MB of places) alone, where it is
// smaller: a pool has as many slots as the memory has room for.
int64_t hash_places(int64_t tokens) {
  int64_t n = 1;
  while (n < 2 * tokens) n *= 2;
  return n;
}
bool by_hash(int64_t tokens, int64_t n_slots) { return n_slots > 1 << 24 && 2 * hash_places(tokens) < n_slots; }

// The place of a slot: in a table by hash the first one from the hash on that has its key, or none.
template <bool kEnter>
__device__ __forceinline__ int32_t* owner_place(const IoArgs& a, int slot) {
  if (a.key == nullptr) return a.owner + slot;
  const uint32_t last = ~0u >> a.hash_shift;
  uint32_t at = (uint32_t)slot * 0x9E3779B1u >> a.hash_shift;  // (2^32 over the golden ratio: neighbours lie far apart)
  for (;; at = (at + 1) & last) {
    const int there = kEnter ? atomicCAS(a.key + at, -1, slot) : a.key[at];
    if (there == slot || there < 0) return a.owner + at;
  }
}
__global__ void __launch_bounds__(256) owner_clear_kernel(IoArgs a) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  ptx::grid_dependency_wait();
  if (a.key) {
    if (i <= ~0u >> a.hash_shift) a.key[i] = a.owner[i] = -1;
  } else if (i < a.tokens) {
    const int slot = a.slots[i];
    if (slot >= 0 && slot < a.n_slots) a.owner[slot] = -1;
  }
}
__global__ void __launch_bounds__(256) owner_claim_kernel(IoArgs a) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  ptx::grid_dependency_wait();
  if (i >= a.tokens) return;
  const int slot = a.slots[i];
  if (slot >= 0 && slot < a.n_slots) atomicMax(owner_place<true>(a, slot), (int)i);
}

// Where the CTA's tokens are: element offsets of their rows in k and v, and the byte offset of head 0's page and the place in it
// (negative: left out).
struct Tile {
  int64_t k[kTile], v[kTile], page[kTile];
  int at[kTile];
};

__device__ __forceinline__ int token_of(const IoArgs& a, int row) { return a.Nk == 1 ? row : (int)__umulhi((uint32_t)row, a.per_head); }

// One thread per token; that a later token names the same slot all of the CTA look for, in one pass over the list.
template <int D, bool kWrite>
__device__ __forceinline__ void find_tokens(const IoArgs& a, Tile& tile, int first, int n) {
  __shared__ int own[kTile], later[kTile];
  if (kWrite && a.owner == nullptr) {  // a slot that several tokens name keeps the last one's values
    int j = first + 1 + threadIdx.x, slot = j < a.tokens ? a.slots[j] : -1;  // (requested together with the CTA's own)
    if (threadIdx.x < n) {
      own[threadIdx.x] = a.slots[first + threadIdx.x];
      later[threadIdx.x] = 0;
    }
    __syncthreads();
    for (; j < a.tokens; j += kIoThreads, slot = j < a.tokens ? a.slots[j] : -1) {
      for (int i = 0; i < n; ++i)
        if (own[i] == slot && first + i < j) later[i] = 1;
    }
    __syncthreads();
  }
  if (threadIdx.x < n) {
    const int tok = first + threadIdx.x;
    int slot = a.slots[tok];
    if (slot >= a.n_slots) {
      if (a.status) atomicCAS(a.status, 0, kStatusBadSlot);
      slot = -1;
    }
    if (kWrite && slot >= 0 && (a.owner ? *owner_place<false>(a, slot) != tok : later[threadIdx.x] != 0)) slot = -1;
    const int b = tok / a.S, s = tok % a.S;
    tile.k[threadIdx.x] = b * a.k.sb + s * a.k.ss;
    tile.v[threadIdx.x] = b * a.v.sb + s * a.v.ss;
    tile.page[threadIdx.x] = (int64_t)(max(slot, 0) / kPage) * a.Nk * Layout<D>::kBytes;
    tile.at[threadIdx.x] = slot < 0 ? -1 : slot % kPage;
  }
  __syncthreads();
}

// The floor is the read (4 D bytes a token and head in bf16) and what is held.  Bound by the wait for the loads, at 21 warps to an SM, and by
// the arithmetic of quantising, 60 % of the ALU pipe.  Every token of 4 prompts of 100 documents, 8 heads of 128: 71 us, its bytes 52; in fp32
// 114 and 92; with a warp to a row and one channel at a time 199.
// Eight lanes take two rows (a token's key and value in one head).  K: four lanes a row, lane t the channels 32 j + 8 t + 0..7, its
// codes one access.  V: all eight both rows, lane g the channels 32 j + 4 g + 0..3.  Each lane makes one scale of either
// and hands its reciprocal round.
template <typename T, int D>
__global__ void __launch_bounds__(kIoThreads) cache_write_kernel(IoArgs a) {
  using L = Layout<D>;
  constexpr int kG = L::kGroups;
  __shared__ Tile tile;
  const int first = blockIdx.x * a.tile, n = min(a.tile, a.tokens - first);
  ptx::grid_dependency_wait();
  find_tokens<D, true>(a, tile, first, n);
  const int lane = threadIdx.x & 31, o = lane & 7, t = lane & 3;
  const bool second = lane & 4;  // K: the octet's second row
  const int rows = n * a.Nk;
  for (int row0 = threadIdx.x / 32 * 8; row0 < rows; row0 += kIoThreads / 4) {
    int at[2], tok[2], head[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = row0 + (lane >> 3) * 2 + x, r = min(row, rows - 1);
      tok[x] = token_of(a, r);
      head[x] = r - tok[x] * a.Nk;
      at[x] = row < rows ? tile.at[tok[x]] : -1;
    }
    if (!__any_sync(0xffffffffu, at[0] >= 0 || at[1] >= 0)) continue;
    const int at_k = second ? at[1] : at[0], tok_k = second ? tok[1] : tok[0], head_k = second ? head[1] : head[0];
    Raw<T, 8> k[kG];
    Raw<T, 4> v[2][kG];
    {
      const T* p = reinterpret_cast<const T*>(a.k.ptr) + tile.k[tok_k] + head_k * a.k.sh + 8 * t;
#pragma unroll
      for (int j = 0; j < kG; ++j) k[j].fetch(p + 32 * j, at_k >= 0);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const T* p = reinterpret_cast<const T*>(a.v.ptr) + tile.v[tok[x]] + head[x] * a.v.sh + 4 * o;
#pragma unroll
      for (int j = 0; j < kG; ++j) v[x][j].fetch(p + 32 * j, at[x] >= 0);
    }
    // ---- scales: this lane's are K's group t mod kG of its row, and V's group o mod kG of row o / kG mod 2 ----
    uint32_t top[kG], top_k = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < kG; ++j) top[j] = k[j].largest();
    reduce_largest<T, kG, 4>(top);
#pragma unroll
    for (int j = 0; j < kG; ++j) top_k = t % kG == j ? top[j] : top_k;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int j = 0; j < kG; ++j) top[j] = v[x][j].largest();
      reduce_largest<T, kG, 8>(top);
#pragma unroll
      for (int j = 0; j < kG; ++j) top_v = o % (2 * kG) == x * kG + j ? top[j] : top_v;
    }
    const float sk = group_scale<T>(top_k), sv = group_scale<T>(top_v);
    const float rk = sk > 0.f ? reciprocal(sk) : 0.f, rv = sv > 0.f ? reciprocal(sv) : 0.f;
    bool divide = (sk > 0.f && (sk < 0x1p-100f || sk > 0x1p100f)) || (sv > 0.f && (sv < 0x1p-100f || sv > 0x1p100f));
    // ---- codes ----
    uint32_t wk[kG], wv[2][kG];
#pragma unroll
    for (int j = 0; j < kG; ++j) wk[j] = quantise(k[j], __shfl_sync(0xffffffffu, rk, (lane & ~3) + j), divide);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int j = 0; j < kG; ++j) wv[x][j] = quantise(v[x][j], __shfl_sync(0xffffffffu, rv, (lane & ~7) + x * kG + j), divide);
    if (__any_sync(0xffffffffu, divide)) {
#pragma unroll
      for (int j = 0; j < kG; ++j) wk[j] = quantise_exactly(k[j], __shfl_sync(0xffffffffu, sk, (lane & ~3) + j));
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < kG; ++j) wv[x][j] = quantise_exactly(v[x][j], __shfl_sync(0xffffffffu, sv, (lane & ~7) + x * kG + j));
    }
    if (at_k >= 0) {
      unsigned char* const p = a.pages + tile.page[tok_k] + (int64_t)head_k * L::kBytes;
      if constexpr (kG == 4) *reinterpret_cast<uint4*>(p + L::k_word(at_k, 0, t)) = make_uint4(wk[0], wk[1], wk[2], wk[3]);
      else *reinterpret_cast<uint2*>(p + L::k_word(at_k, 0, t)) = make_uint2(wk[0], wk[1]);
      if (t < kG) *reinterpret_cast<__nv_bfloat16*>(p + L::k_scale(at_k, t)) = __float2bfloat16_rn(sk);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (at[x] < 0) continue;
      unsigned char* const p = a.pages + tile.page[tok[x]] + (int64_t)head[x] * L::kBytes;
      uint32_t w[kG / 2];
#pragma unroll
      for (int j = 0; j < kG; j += 2) w[j / 2] = rotl(__byte_perm(wv[x][j], wv[x][j + 1], 0x5410), 3);
      if constexpr (kG == 4) *reinterpret_cast<uint2*>(p + L::v_word(at[x], o, 0)) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(p + L::v_word(at[x], o, 0)) = w[0];
      if (o / kG == x) *reinterpret_cast<__nv_bfloat16*>(p + L::v_scale(at[x], o % kG)) = __float2bfloat16_rn(sv);
    }
  }
}

// four values as bf16 -> memory
__device__ __forceinline__ void write4(__nv_bfloat16* p, uint2 x) { __stcs(reinterpret_cast<uint2*>(p), x); }
__device__ __forceinline__ void write4(float* p, uint2 x) {
  __stcs(reinterpret_cast<float4*>(p), make_float4(bf_lo(x.x), bf_hi(x.x), bf_lo(x.y), bf_hi(x.y)));
}
__device__ __forceinline__ void write8(__nv_bfloat16* p, uint2 x, uint2 y) { __stcs(reinterpret_cast<uint4*>(p), make_uint4(x.x, x.y, y.x, y.y)); }
__device__ __forceinline__ void write8(float* p, uint2 x, uint2 y) {
  write4(p, x);
  write4(p + 4, y);
}

// Bound by the writes: 4 prompts of 100 documents of 32 to 256 tokens in bf16 60 us, 93 % of the copy bandwidth (a lane's stores 16 bytes; with a
// warp to a row 99); in fp32 133, 76 %.  Lanes as in the write.
template <typename T, int D>
__global__ void __launch_bounds__(kIoThreads) cache_read_kernel(IoArgs a) {
  using L = Layout<D>;
  constexpr int kG = L::kGroups;
  __shared__ Tile tile;
  const int first = blockIdx.x * a.tile, n = min(a.tile, a.tokens - first);
  ptx::grid_dependency_wait();
  find_tokens<D, false>(a, tile, first, n);
  const int lane = threadIdx.x & 31, o = lane & 7, t = lane & 3;
  const bool second = lane & 4;
  const int rows = n * a.Nk;
  const Codes codes = a.codes;
#pragma unroll 2
  for (int row0 = threadIdx.x / 32 * 8 + (lane >> 3) * 2; row0 < rows; row0 += kIoThreads / 4) {
    int at[2], tok[2], head[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int row = min(row0 + x, rows - 1);  // (the last row of an odd number is written twice, the same both times)
      tok[x] = token_of(a, row);
      head[x] = row - tok[x] * a.Nk;
      at[x] = tile.at[tok[x]];
    }
    const int at_k = second ? at[1] : at[0], tok_k = second ? tok[1] : tok[0], head_k = second ? head[1] : head[0];
    uint32_t wk[kG] = {}, sk[kG / 2] = {}, wv[2][kG / 2] = {}, sv[2][kG] = {};  // (a scale of 0: zeros)
    if (at_k >= 0) {
      const unsigned char* const p = a.pages + tile.page[tok_k] + (int64_t)head_k * L::kBytes;
      load_words<D>(p + L::k_word(at_k, 0, t), wk);
      load_scales<D>(p + L::k_scale(at_k, 0), sk);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (at[x] < 0) continue;
      const unsigned char* const p = a.pages + tile.page[tok[x]] + (int64_t)head[x] * L::kBytes;
      load_scales<D>(p + L::v_word(at[x], o, 0), wv[x]);  // (as many words)
      load_words<D>(p + L::v_scale(at[x] & ~1, 0), sv[x]);  // both tokens' of the pair
    }
    T* const pk = reinterpret_cast<T*>(a.k.ptr) + tile.k[tok_k] + head_k * a.k.sh + 8 * t;
#pragma unroll
    for (int j = 0; j < kG; ++j) {
      const Pairs p = pairs_of(codes, wk[j], __byte_perm(sk[j / 2], 0, j % 2 ? 0x3232 : 0x1010));
      write8(pk + 32 * j, low_values(p), high_values(p));
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      T* const pv = reinterpret_cast<T*>(a.v.ptr) + tile.v[tok[x]] + head[x] * a.v.sh + 4 * o;
#pragma unroll
      for (int j = 0; j < kG; j += 2) {  // the low half of a word is group j's, the high one j + 1's
        const Pairs p = pairs_of(codes, rotr(wv[x][j / 2], 3), __byte_perm(sv[x][j], sv[x][j + 1], at[x] & 1 ? 0x7632 : 0x5410));
        write4(pv + 32 * j, low_values(p));
        write4(pv + 32 * j + 32, high_values(p));
      }
    }
  }
}

IoArgs make_args(const brk_cache& c, const brk_view& k, const brk_view& v, int B, int S, const int32_t* slots, int32_t* status) {
  IoArgs a;
  a.pages = static_cast<unsigned char*>(c.pages);
  a.k = make_view(k);
  a.v = make_view(v);
  a.slots = slots;
  a.owner = a.key = nullptr;
  a.hash_shift = 0;
  a.status = status;
  a.n_slots = (int64_t)c.n_pages * kPage;
  a.tokens = B * S;
  a.S = S;
  a.Nk = c.Nk;
  a.per_head = (uint32_t)(((1ull << 32) + c.Nk - 1) / c.Nk);
  // Tokens of a CTA: those that make it two CTAs an SM, at most as many as give a warp four rounds.  (bf16, 8 heads of 128; of 592 CTAs 512
  // tokens took 4.9 us, now 3.4; 1024 7.7 and 4.2, 16384 24.1 and 23.1; of 148 CTAs 512 3.5, 1024 5.0.)
  const int most = std::min(kTile, std::max(1, kIoThreads / a.Nk)), ctas = 2 * std::max(1, sm_count());
  a.tile = std::min(most, (int)((a.tokens + (int64_t)ctas - 1) / ctas));
  return a;
}
dim3 grid_of(const IoArgs& a) { return dim3((unsigned)((a.tokens + (int64_t)a.tile - 1) / a.tile)); }

}  // namespace

size_t cache_write_workspace(const brk_cache& c, int B, int S) {
  const int64_t tokens = (int64_t)B * S, n_slots = (int64_t)c.n_pages * kPage;
  if (tokens <= kScan) return 0;
  return sizeof(int32_t) * (by_hash(tokens, n_slots) ? 2 * hash_places(tokens) : n_slots);
}

int cache_write_launch(int dtype, const brk_cache& c, const brk_view& k, const brk_view& v, int B, int S, const int32_t* slots, void* ws,
                       int32_t* status, cudaStream_t st) {
  IoArgs a = make_args(c, k, v, B, S, slots, status);
  if (a.tokens > kScan) {
    a.owner = static_cast<int32_t*>(ws);
    int64_t cleared = a.tokens;
    if (by_hash(a.tokens, a.n_slots)) {
      cleared = hash_places(a.tokens);
      a.key = a.owner + cleared;
      for (a.hash_shift = 32; (int64_t)1 << (32 - a.hash_shift) < cleared;) --a.hash_shift;
    }
    auto of = [](int64_t n) { return dim3((unsigned)((n + 255) / 256)); };
    int rc = launch_dependent(owner_clear_kernel, of(cleared), dim3(256), 0, st, a);
    if (rc || (rc = launch_dependent(owner_claim_kernel, of(a.tokens), dim3(256), 0, st, a))) return rc;
  }
  auto run = [&](auto kern) { return launch_dependent(kern, grid_of(a), dim3(kIoThreads), 0, st, a); };
  if (dtype == BRK_BF16) return c.D == 128 ? run(cache_write_kernel<__nv_bfloat16, 128>) : run(cache_write_kernel<__nv_bfloat16, 64>);
  return c.D == 128 ? run(cache_write_kernel<float, 128>) : run(cache_write_kernel<float, 64>);
}

int cache_read_launch(int dtype, const brk_cache& c, const brk_view& k, const brk_view& v, int B, int S, const int32_t* slots,
                      int32_t* status, cudaStream_t st) {
  const IoArgs a = make_args(c, k, v, B, S, slots, status);
  auto run = [&](auto kern) { return launch_dependent(kern, grid_of(a), dim3(kIoThreads), 0, st, a); };
  if (dtype == BRK_BF16) return c.D == 128 ? run(cache_read_kernel<__nv_bfloat16, 128>) : run(cache_read_kernel<__nv_bfloat16, 64>);
  return c.D == 128 ? run(cache_read_kernel<float, 128>) : run(cache_read_kernel<float, 64>);
}

}  // namespace brk
