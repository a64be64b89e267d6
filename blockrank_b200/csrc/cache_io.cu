// The 4-bit cache: quantising keys and values as they are written, and reading them back.
//
// s = max|x| / 7 of a group of 32 channels, rounded to 5 significant bits (nearest, ties to even; never to a finer quantum than
// 2^-130; at most 1.9375 * 2^122), n = round(x / s) (ties to even) within -7..7.  Rounding s to the nearest never cuts the
// largest value off: 7 / (1 - 2^-5) < 7.5.
// Both decisions are those of exact arithmetic, with one 32-bit division each.  A border of n is (k + 1/2) s, 4 bits times 5; of
// s, a 6-bit number times 7: representable, so a 32-bit x is either equal to it or off by more than half a last place of the
// quotient, and the correctly rounded quotient lies on the border only if x does.
#include <algorithm>

#include "cache_layout.cuh"

namespace brk {
namespace {

using namespace cache;

struct IoArgs {
  unsigned char* pages;
  View k, v;
  const int32_t* slots;
  int32_t* owner;  // [slots of the pool]: the last token of the call that names the slot; null: looked up in `slots`
  int32_t* status;
  int64_t n_slots;
  int64_t tokens;  // B S
  int S, Nk;
};

// s of a group with this largest magnitude; NaN where the group holds NaN or an infinity
__device__ __forceinline__ float group_scale(float amax) {
  if (!(amax < INFINITY)) return __uint_as_float(0x7FC00000u);
  const uint32_t b = __float_as_uint(__fdiv_rn(amax, 7.f));
  const float s = __uint_as_float((b + 0x3FFFFu + ((b >> 19) & 1u)) & ~0x7FFFFu);
  return fminf(s, 1.9375f * 5316911983139663491615228241121378304.f);  // 2^122
}

__device__ __forceinline__ uint32_t code_of(float x, float s) {
  const float n = rintf(__fdiv_rn(x, s));
  return (uint32_t)((int)fminf(fmaxf(n, -7.f), 7.f) + 8);
}

// 8 channels of a lane -> their codes, channel i in bits 4 i .. 4 i + 3; the group is the 4 lanes of a quad
__device__ __forceinline__ uint32_t quantise(const float (&x)[8], float& s) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = isnan(x[i]) ? INFINITY : fmaxf(amax, fabsf(x[i]));
  // (a NaN has become an infinity, which fmaxf keeps)
#pragma unroll
  for (int off = 1; off <= 2; off <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, off));
  s = group_scale(amax);
  uint32_t w = 0x88888888u;
  if (s > 0.f) {
    w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= code_of(x[i], s) << (4 * i);
  }
  return w;
}

constexpr int kIoThreads = 256;
// Calls with at most this many tokens look for a later token with the same slot in the list itself; others go through `owner`.
constexpr int kScan = 1024;

__global__ void __launch_bounds__(256) owner_clear_kernel(const int32_t* slots, int64_t tokens, int64_t n_slots, int32_t* owner) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < tokens && slots[i] >= 0 && slots[i] < n_slots) owner[slots[i]] = -1;
}
__global__ void __launch_bounds__(256) owner_claim_kernel(const int32_t* slots, int64_t tokens, int64_t n_slots, int32_t* owner) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i < tokens && slots[i] >= 0 && slots[i] < n_slots) atomicMax(owner + slots[i], (int32_t)i);
}

// D / 8 lanes per (token, head), 8 channels each.
template <typename T, int D>
__global__ void __launch_bounds__(kIoThreads) cache_write_kernel(IoArgs a) {
  using L = Layout<D>;
  constexpr int kLanes = D / 8;
  const int64_t row = ((int64_t)blockIdx.x * kIoThreads + threadIdx.x) / kLanes;
  const int l = threadIdx.x % kLanes, j = l / 4, t = l % 4;
  const int64_t tok = row / a.Nk;
  const int h = (int)(row % a.Nk);
  int slot = tok < a.tokens ? a.slots[tok] : -1;
  if (slot >= a.n_slots) {
    if (l == 0 && h == 0 && a.status) atomicCAS(a.status, 0, kStatusBadSlot);
    slot = -1;
  }
  // a slot that several tokens name keeps the last one's values
  bool later = false;
  if (slot >= 0 && a.owner) {
    later = a.owner[slot] != (int32_t)tok;
  } else if (slot >= 0) {
    for (int64_t i = tok + 1 + l; i < a.tokens; i += kLanes) later |= a.slots[i] == slot;
  }
  const unsigned mine = ((1u << kLanes) - 1) << (threadIdx.x % 32 / kLanes * kLanes);
  if (__ballot_sync(0xffffffffu, later) & mine) slot = -1;
  float x[8] = {}, y[8] = {};
  if (slot >= 0) {
    const int64_t b = tok / a.S, s = tok % a.S;
    load8(reinterpret_cast<const T*>(a.k.ptr) + b * a.k.sb + h * a.k.sh + s * a.k.ss + 8 * l, x);
    load8(reinterpret_cast<const T*>(a.v.ptr) + b * a.v.sb + h * a.v.sh + s * a.v.ss + 8 * l, y);
  }
  float sk, sv;
  const uint32_t wk = quantise(x, sk), wv = quantise(y, sv);
  // V: channels 4 g + 0..3 of groups 2 w and 2 w + 1 share a word; this lane has g = 2 t and 2 t + 1 of group j, its partner 4
  // lanes on those of group j ^ 1.  Even groups store g = 2 t, odd ones 2 t + 1.
  const uint32_t other = __shfl_xor_sync(0xffffffffu, wv, 4);
  const uint32_t word = (j & 1) ? __byte_perm(other, wv, 0x7632) : __byte_perm(wv, other, 0x5410);
  if (slot < 0) return;
  unsigned char* const page = a.pages + ((int64_t)(slot / kPage) * a.Nk + h) * L::kBytes;
  const int at = slot % kPage;
  *reinterpret_cast<uint32_t*>(page + L::k_word(at, j, t)) = wk;
  *reinterpret_cast<uint32_t*>(page + L::v_word(at, 2 * t + (j & 1), j >> 1)) = rotl(word, 3);
  if (t == 0) *reinterpret_cast<__nv_bfloat16*>(page + L::k_scale(at, j)) = __float2bfloat16_rn(sk);
  if (t == 1) *reinterpret_cast<__nv_bfloat16*>(page + L::v_scale(at, j)) = __float2bfloat16_rn(sv);
}

template <typename T, int D>
__global__ void __launch_bounds__(kIoThreads) cache_read_kernel(IoArgs a) {
  using L = Layout<D>;
  constexpr int kLanes = D / 8;
  const int64_t row = ((int64_t)blockIdx.x * kIoThreads + threadIdx.x) / kLanes;
  const int l = threadIdx.x % kLanes, j = l / 4, t = l % 4;
  const int64_t tok = row / a.Nk;
  const int h = (int)(row % a.Nk);
  if (tok >= a.tokens) return;
  int slot = a.slots[tok];
  if (slot >= a.n_slots) {
    if (l == 0 && h == 0 && a.status) atomicCAS(a.status, 0, kStatusBadSlot);
    slot = -1;
  }
  float x[8] = {}, y[8] = {};
  if (slot >= 0) {
    const unsigned char* const page = a.pages + ((int64_t)(slot / kPage) * a.Nk + h) * L::kBytes;
    const int at = slot % kPage;
    const uint32_t wk = *reinterpret_cast<const uint32_t*>(page + L::k_word(at, j, t));
    const uint32_t w0 = rotr(*reinterpret_cast<const uint32_t*>(page + L::v_word(at, 2 * t, j >> 1)), 3);
    const uint32_t w1 = rotr(*reinterpret_cast<const uint32_t*>(page + L::v_word(at, 2 * t + 1, j >> 1)), 3);
    const uint32_t wv = __byte_perm(w0, w1, (j & 1) ? 0x7632 : 0x5410);
    const float sk = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(page + L::k_scale(at, j)));
    const float sv = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(page + L::v_scale(at, j)));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = (float)((int)((wk >> (4 * i)) & 15u) - 8) * sk;
      y[i] = (float)((int)((wv >> (4 * i)) & 15u) - 8) * sv;
    }
  }
  const int64_t b = tok / a.S, s = tok % a.S;
  store8(reinterpret_cast<T*>(a.k.ptr) + b * a.k.sb + h * a.k.sh + s * a.k.ss + 8 * l, x);
  store8(reinterpret_cast<T*>(a.v.ptr) + b * a.v.sb + h * a.v.sh + s * a.v.ss + 8 * l, y);
}

IoArgs make_args(const brk_cache& c, const brk_view& k, const brk_view& v, int B, int S, const int32_t* slots, int32_t* status) {
  IoArgs a;
  a.pages = static_cast<unsigned char*>(c.pages);
  a.k = make_view(k);
  a.v = make_view(v);
  a.slots = slots;
  a.owner = nullptr;
  a.status = status;
  a.n_slots = (int64_t)c.n_pages * kPage;
  a.tokens = (int64_t)B * S;
  a.S = S;
  a.Nk = c.Nk;
  return a;
}
unsigned blocks_for(const IoArgs& a, int D) { return (unsigned)((a.tokens * a.Nk * (D / 8) + kIoThreads - 1) / kIoThreads); }

}  // namespace

size_t cache_write_workspace(const brk_cache& c, int B, int S) {
  return (int64_t)B * S <= kScan ? 0 : (size_t)c.n_pages * kPage * sizeof(int32_t);
}

int cache_write_launch(int dtype, const brk_cache& c, const brk_view& k, const brk_view& v, int B, int S, const int32_t* slots, void* ws,
                       int32_t* status, cudaStream_t st) {
  IoArgs a = make_args(c, k, v, B, S, slots, status);
  if (a.tokens > kScan) {
    a.owner = static_cast<int32_t*>(ws);
    const unsigned n = (unsigned)((a.tokens + 255) / 256);
    owner_clear_kernel<<<n, 256, 0, st>>>(slots, a.tokens, a.n_slots, a.owner);
    BRK_LAUNCHED();
    owner_claim_kernel<<<n, 256, 0, st>>>(slots, a.tokens, a.n_slots, a.owner);
    BRK_LAUNCHED();
  }
  const unsigned n = blocks_for(a, c.D);
  if (dtype == BRK_BF16) {
    if (c.D == 128) cache_write_kernel<__nv_bfloat16, 128><<<n, kIoThreads, 0, st>>>(a);
    else cache_write_kernel<__nv_bfloat16, 64><<<n, kIoThreads, 0, st>>>(a);
  } else {
    if (c.D == 128) cache_write_kernel<float, 128><<<n, kIoThreads, 0, st>>>(a);
    else cache_write_kernel<float, 64><<<n, kIoThreads, 0, st>>>(a);
  }
  BRK_LAUNCHED();
  return BRK_OK;
}

int cache_read_launch(int dtype, const brk_cache& c, const brk_view& k, const brk_view& v, int B, int S, const int32_t* slots,
                      int32_t* status, cudaStream_t st) {
  const IoArgs a = make_args(c, k, v, B, S, slots, status);
  const unsigned n = blocks_for(a, c.D);
  if (dtype == BRK_BF16) {
    if (c.D == 128) cache_read_kernel<__nv_bfloat16, 128><<<n, kIoThreads, 0, st>>>(a);
    else cache_read_kernel<__nv_bfloat16, 64><<<n, kIoThreads, 0, st>>>(a);
  } else {
    if (c.D == 128) cache_read_kernel<float, 128><<<n, kIoThreads, 0, st>>>(a);
    else cache_read_kernel<float, 64><<<n, kIoThreads, 0, st>>>(a);
  }
  BRK_LAUNCHED();
  return BRK_OK;
}

}  // namespace brk
