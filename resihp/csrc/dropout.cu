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
#include "common.cuh"
#include "launch.h"

namespace resihp {

namespace {

__device__ __forceinline__ uint4 philox(uint4 c, uint2 k) {
  #pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = uint64_t(c.x) * 0xD2511F53u, b = uint64_t(c.z) * 0xCD9E8D57u;
    c = make_uint4(uint32_t(b >> 32) ^ c.y ^ k.x, uint32_t(b), uint32_t(a >> 32) ^ c.w ^ k.y, uint32_t(a));
    k.x += 0x9E3779B9u;
    k.y += 0xBB67AE85u;
  }
  return c;
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
  const void* residual;  // nullptr: none
  void* out;
  int64_t n;             // elements
  int64_t first;         // logical index of element 0
  uint64_t seed, offset;
  const int64_t* state;  // device (seed, offset), nullptr: the two values above
  uint32_t drop;
  float scale;
};

// One thread per Philox block. VEC: element 0 starts a block and the pointers are 16-byte
// aligned, so whole blocks move as vectors; otherwise (and for a cut block at either end)
// element by element.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs a) {
  pdl_enter();
  const T* x = static_cast<const T*>(a.x);
  const T* res = static_cast<const T*>(a.residual);
  T* out = static_cast<T*>(a.out);
  uint64_t seed = a.seed, offset = a.offset;
  if (a.state != nullptr) {
    seed = uint64_t(a.state[0]);
    offset = uint64_t(a.state[1]);
  }
  const uint64_t b0 = uint64_t(a.first) >> 3;
  const uint64_t blocks = ((uint64_t(a.first) + uint64_t(a.n) + 7) >> 3) - b0;
  for (uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < blocks; i += uint64_t(gridDim.x) * blockDim.x) {
    const int64_t at = int64_t((b0 + i) << 3) - a.first;  // position of the block's lane 0 (may be below 0)
    const bool whole = VEC && at + 8 <= a.n;
    Pack8<T> px, pr;
    if (whole) {
      px = *reinterpret_cast<const Pack8<T>*>(x + at);
      if (res != nullptr) pr = *reinterpret_cast<const Pack8<T>*>(res + at);
    }
    const uint64_t b = b0 + i;
    const uint4 r = philox(make_uint4(uint32_t(b), uint32_t(b >> 32), uint32_t(offset), uint32_t(offset >> 32)),
                           make_uint2(uint32_t(seed), uint32_t(seed >> 32)));
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    if (whole) {
      Pack8<T> po;
      #pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t u = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu;
        float v = u >= a.drop ? to_float(px.v[e]) * a.scale : 0.f;
        if (res != nullptr) v += to_float(pr.v[e]);
        po.v[e] = from_float<T>(v);
      }
      *reinterpret_cast<Pack8<T>*>(out + at) = po;
    } else {
      #pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t p = at + e;
        if (p < 0 || p >= a.n) continue;
        const uint32_t u = (e & 1) ? w[e >> 1] >> 16 : w[e >> 1] & 0xFFFFu;
        float v = u >= a.drop ? to_float(x[p]) * a.scale : 0.f;
        if (res != nullptr) v += to_float(res[p]);
        out[p] = from_float<T>(v);
      }
    }
  }
}

template <typename T>
void launch(const DropoutArgs& a, int num_sms, cudaStream_t st) {
  const uintptr_t al = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.residual) |
                       reinterpret_cast<uintptr_t>(a.out);
  const bool vec = al % 16 == 0 && a.first % 8 == 0;
  const int64_t blocks = ((a.first + a.n + 7) >> 3) - (a.first >> 3);
  const int grid = int(std::min<int64_t>((blocks + 255) / 256, int64_t(num_sms) * 16));
  auto kernel = vec ? dropout_kernel<T, true> : dropout_kernel<T, false>;
  RESIHP_CUDA_CHECK(launch_pdl(kernel, grid, 256, 0, st, a));
}

}  // namespace

void dropout(const void* x, const void* residual, void* out, bool bf16, int64_t n, int64_t first, uint64_t seed,
             uint64_t offset, const int64_t* state, uint32_t drop, int num_sms, cudaStream_t st) {
  RESIHP_CHECK(drop <= 65536, "dropout threshold out of range");
  RESIHP_CHECK(first >= 0 && n >= 0 && first <= INT64_MAX - n - 8, "dropout indices pass 63 bits");
  if (n == 0) return;
  DropoutArgs a{x, residual, out, n, first, seed, offset, state, drop,
                drop < 65536 ? 65536.f / float(65536 - drop) : 0.f};
  if (bf16) launch<__nv_bfloat16>(a, num_sms, st);
  else launch<float>(a, num_sms, st);
}

}  // namespace resihp
