// Inverted dropout with a mask that is never stored (no counterpart in the reference,
// whose blocks have no dropout).
//
// Element i of the logical tensor (row-major, first_row rows into it) belongs to block
// b = i / 8 and lane i % 8. Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011) with key = seed and counter = (b, offset) gives
// the block four 32-bit words, i.e. eight 16-bit numbers u (low half of a word first):
//   keep_i = u_i >= drop,   out_i = keep_i ? x_i * 65536 / (65536 - drop) : 0  (+ residual_i)
// with drop = round(65536 p), so the kept share is exact in expectation. Sixteen bits per
// element halve the integer work of one word per element and put p on a grid of 1.5e-5.
// The backward pass runs the same kernel on the output gradient: nothing is kept but the
// seed, and a token shard (first_row) draws its part of the whole tensor's mask.
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace resihp {

namespace {

constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u;
constexpr uint32_t kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;

// The ten rounds' keys.
struct RoundKeys {
  uint32_t x[10], y[10];
};

__host__ __device__ __forceinline__ RoundKeys round_keys(uint64_t seed) {
  RoundKeys k;
  for (int r = 0; r < 10; ++r) {
    k.x[r] = uint32_t(seed) + uint32_t(r) * kPhiloxW0;
    k.y[r] = uint32_t(seed >> 32) + uint32_t(r) * kPhiloxW1;
  }
  return k;
}

__device__ __forceinline__ void philox(uint64_t block, uint64_t offset, const RoundKeys& k, uint32_t (&w)[4]) {
  uint4 c = make_uint4(uint32_t(block), uint32_t(block >> 32), uint32_t(offset), uint32_t(offset >> 32));
  #pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = uint64_t(c.x) * kPhiloxM0, b = uint64_t(c.z) * kPhiloxM1;
    c = make_uint4(uint32_t(b >> 32) ^ c.y ^ k.x[r], uint32_t(b), uint32_t(a >> 32) ^ c.w ^ k.y[r], uint32_t(a));
  }
  w[0] = c.x;
  w[1] = c.y;
  w[2] = c.z;
  w[3] = c.w;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16(v); }

// Eight elements moved as 16-byte vectors.
template <typename T>
struct alignas(16) Pack8 {
  T v[8];
};

struct DropoutArgs {
  const void* x;
  const void* residual;
  void* out;
  int64_t n;             // elements
  int64_t first;         // logical index of element 0
  RoundKeys keys;        // the kernels that read no ``state`` take these two from their constants
  uint64_t offset;
  const int64_t* state;  // device (seed, offset)
  uint32_t last_drop;    // an element is kept if its number, as the high half of a word, is above this
  float scale;
};

// Element e of a block: its number is a half of word e / 2. The high half of w is at least
// ``drop`` exactly if w > (drop << 16) - 1 = last_drop (all ones for drop = 65536: never).
__device__ __forceinline__ bool kept(const uint32_t (&w)[4], int e, uint32_t last_drop) {
  return ((e & 1) ? w[e >> 1] : w[e >> 1] << 16) > last_drop;
}

template <typename T, bool DROP, bool RES>
__device__ __forceinline__ T drop_one(T x, T res, const uint32_t (&w)[4], int e, const DropoutArgs& a) {
  float v = RES ? to_float(res) : 0.f;
  if (!DROP || kept(w, e, a.last_drop)) v = RES ? fmaf(to_float(x), a.scale, v) : to_float(x) * a.scale;
  return from_float<T>(v);
}

// Whole blocks as 16-byte vectors (element 0 starts a block, aligned pointers). A thread takes
// two blocks of a 512-block tile, at fixed distances: one address computation, both loads under
// way during the integer work (twenty 32 x 32 > 64 bit products per block), which adds 14 % to
// the memory's time: ten rounds take 60 us, five would take 55 and none 53 (16384 x 5120 bf16, 335
// MB moved, 5.6 TB/s of the 6.5 a copy reaches). The round keys come from the kernel's constants,
// so a round is two products and two three-way exclusive ors. DROP false (p below 2^-17): nothing
// is drawn.
constexpr int kTile = 512;

template <typename T, bool DROP, bool RES, bool STATE>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutArgs a) {
  pdl_enter();
  RoundKeys own;
  uint64_t offset = a.offset;
  if (STATE) {
    own = round_keys(uint64_t(a.state[0]));
    offset = uint64_t(a.state[1]);
  }
  const RoundKeys& keys = STATE ? own : a.keys;
  const uint64_t b0 = uint64_t(a.first) >> 3;
  const int64_t blocks = a.n >> 3;
  for (int64_t i = int64_t(blockIdx.x) * kTile + threadIdx.x; i < blocks; i += int64_t(gridDim.x) * kTile) {
    const Pack8<T>* x = static_cast<const Pack8<T>*>(a.x) + i;
    const Pack8<T>* res = static_cast<const Pack8<T>*>(a.residual) + i;
    Pack8<T>* out = static_cast<Pack8<T>*>(a.out) + i;
    const bool two = i + kTile / 2 < blocks;
    Pack8<T> px[2], pr[2];
    px[0] = x[0];
    if (RES) pr[0] = res[0];
    if (two) {
      px[1] = x[kTile / 2];
      if (RES) pr[1] = res[kTile / 2];
    }
    #pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u == 1 && !two) break;
      uint32_t w[4];
      if (DROP) philox(b0 + uint64_t(i + u * (kTile / 2)), offset, keys, w);
      Pack8<T> po;
      #pragma unroll
      for (int e = 0; e < 8; ++e) po.v[e] = drop_one<T, DROP, RES>(px[u].v[e], pr[u].v[e], w, e, a);
      out[u * (kTile / 2)] = po;
    }
  }
  // the elements behind the last whole block
  const int64_t p = (blocks << 3) + threadIdx.x;
  if (blockIdx.x == 0 && p < a.n) {
    uint32_t w[4];
    if (DROP) philox(b0 + uint64_t(blocks), offset, keys, w);
    const T r = RES ? static_cast<const T*>(a.residual)[p] : from_float<T>(0.f);
    static_cast<T*>(a.out)[p] = drop_one<T, DROP, RES>(static_cast<const T*>(a.x)[p], r, w, int(threadIdx.x), a);
  }
}

// Any alignment and any place of element 0 in its block: one block per thread, element by element.
template <typename T, bool DROP, bool RES, bool STATE>
__global__ void __launch_bounds__(256) dropout_any_kernel(const __grid_constant__ DropoutArgs a) {
  pdl_enter();
  RoundKeys own;
  uint64_t offset = a.offset;
  if (STATE) {
    own = round_keys(uint64_t(a.state[0]));
    offset = uint64_t(a.state[1]);
  }
  const RoundKeys& keys = STATE ? own : a.keys;
  const uint64_t b0 = uint64_t(a.first) >> 3;
  const uint64_t blocks = ((uint64_t(a.first) + uint64_t(a.n) + 7) >> 3) - b0;
  for (uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < blocks; i += uint64_t(gridDim.x) * blockDim.x) {
    const int64_t at = int64_t((b0 + i) << 3) - a.first;  // position of the block's lane 0 (may be below 0)
    uint32_t w[4];
    if (DROP) philox(b0 + i, offset, keys, w);
    T x[8], r[8];
    #pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = at + e >= 0 && at + e < a.n;
      x[e] = in ? static_cast<const T*>(a.x)[at + e] : from_float<T>(0.f);
      r[e] = RES && in ? static_cast<const T*>(a.residual)[at + e] : from_float<T>(0.f);
    }
    #pragma unroll
    for (int e = 0; e < 8; ++e)
      if (at + e >= 0 && at + e < a.n) static_cast<T*>(a.out)[at + e] = drop_one<T, DROP, RES>(x[e], r[e], w, e, a);
  }
}

template <typename T, bool DROP, bool RES, bool STATE>
void launch_as(const DropoutArgs& a, int num_sms, cudaStream_t st) {
  const uintptr_t al = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.residual) |
                       reinterpret_cast<uintptr_t>(a.out);
  const bool vec = al % 16 == 0 && a.first % 8 == 0;
  const int64_t work = (a.n + 14) / 8;  // blocks touched, at most
  const int64_t per = vec ? kTile : 256;
  const int grid = int(std::min<int64_t>((work + per - 1) / per, int64_t(num_sms) * 16));
  auto kernel = vec ? dropout_kernel<T, DROP, RES, STATE> : dropout_any_kernel<T, DROP, RES, STATE>;
  RESIHP_CUDA_CHECK(launch_pdl(kernel, grid, 256, 0, st, a));
}

template <typename T, bool DROP, bool RES>
void launch_as(const DropoutArgs& a, int num_sms, cudaStream_t st) {
  if (DROP && a.state != nullptr) launch_as<T, DROP, RES, DROP>(a, num_sms, st);
  else launch_as<T, DROP, RES, false>(a, num_sms, st);
}

template <typename T>
void launch(const DropoutArgs& a, bool drop, int num_sms, cudaStream_t st) {
  if (a.residual != nullptr) {
    if (drop) launch_as<T, true, true>(a, num_sms, st);
    else launch_as<T, false, true>(a, num_sms, st);
  } else {
    if (drop) launch_as<T, true, false>(a, num_sms, st);
    else launch_as<T, false, false>(a, num_sms, st);
  }
}

}  // namespace

void dropout(const void* x, const void* residual, void* out, bool bf16, int64_t n, int64_t first, uint64_t seed,
             uint64_t offset, const int64_t* state, uint32_t drop, int num_sms, cudaStream_t st) {
  RESIHP_CHECK(drop <= 65536, "dropout threshold out of range");
  RESIHP_CHECK(first >= 0 && n >= 0 && first <= INT64_MAX - n - 8, "dropout indices pass 63 bits");
  if (n == 0) return;
  const DropoutArgs a{x, residual, out, n, first, round_keys(seed), offset, state, (drop << 16) - 1u,
                      drop < 65536 ? 65536.f / float(65536 - drop) : 0.f};
  if (bf16) launch<__nv_bfloat16>(a, drop != 0, num_sms, st);
  else launch<float>(a, drop != 0, num_sms, st);
}

}  // namespace resihp
