// Routing of a sparse (mixture-of-experts) MLP around its per-expert products (no
// counterpart in the reference, whose blocks are dense): the router's choice of experts,
// the plan that sorts the (token, choice) pairs by expert, and the two row movements.
//
//   route     ids[t, j] = the expert of token t's j-th largest logit (lowest index first
//             among equal ones), weights = softmax over all experts or over the chosen ones
//   plan      offsets[e] = pairs of the experts before e;  slots[t, j] = the pair's place in
//             the order (expert, token, choice); pairs of no expert go behind offsets[E]
//   scatter   y[slots[t, j]] = w[t, j] x[t]                (dispatch; combine's gradient)
//   gather    out[t] = residual[t] + sum_j w[t, j] y[slots[t, j]]   (combine; dispatch's)
//
// The plan is a stable counting sort in two launches: the first counts experts per run of
// consecutive pairs, the second adds up the counts of the runs before its own, ranks its
// pairs warp by warp and writes their places. Nothing is decided by the order of atomics
// (they only count), so a plan is the same on every run; and no state outlives a call.
//
// Both row movements go token by token, so a token's row is read (or written) once however
// many experts it has: k + 1 rows move per token, which is all that has to move.
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace resihp {

namespace {

// ---- routing --------------------------------------------------------------------------

// A row's logits in registers: 32 per lane leave room for half the warps.
template <int VPT>
constexpr int kRouteThreads = VPT > 8 ? 512 : 1024;
constexpr int kBwdThreads = 256;

// Unsigned order of the floats, both zeros alike, NaN above all, never 0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
constexpr uint32_t kKeyNone = 0x007FFFFFu;  // order_key(-inf); anything up to it is not allowed

__device__ __forceinline__ float logit_at(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float logit_at(const float* p) { return *p; }
__device__ __forceinline__ void store_logit(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }

__device__ __forceinline__ float key_value(uint32_t key) {
  if (key == 0xFFFFFFFFu) return __uint_as_float(0x7FFFFFFFu);
  return __uint_as_float((key & 0x80000000u) ? key & 0x7FFFFFFFu : ~key);
}

// LPR lanes share a row, lane l holds the logits l, l + LPR, ... Choice j ends up on lane j.
// A choice is the largest key, then the lowest index that has it: two warp reductions on whole
// warps, shuffles within the parts of a shared one.
template <typename T, int LPR, int VPT>
__global__ void __launch_bounds__(kRouteThreads<VPT>) route_kernel(const T* __restrict__ logits, int64_t ld, int tokens,
                                                              int experts, int k, bool normalize, int rows_per_block,
                                                              float* __restrict__ weights, int* __restrict__ ids,
                                                              int* __restrict__ counts) {
  pdl_enter();
  extern __shared__ int hist[];  // [experts + 1]
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  constexpr int kRows = kRouteThreads<VPT> / LPR;
  const int sub = threadIdx.x / LPR, lane = threadIdx.x % LPR;
  const int first = blockIdx.x * rows_per_block;
  const int last = min(tokens, first + rows_per_block);
  // whole warps walk together (the reductions need every lane); rows past the end are idle
  float ahead[VPT];  // the next row's logits, on their way during this row's reductions
  auto fetch = [&](int row) {
    #pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int e = lane + v * LPR;
      ahead[v] = row < last && e < experts ? logit_at(logits + int64_t(row) * ld + e) : -INFINITY;
    }
  };
  fetch(first + sub);
  for (int base = first; base < last; base += kRows) {
    const int row = base + sub;
    const bool live = row < last;
    float x[VPT];
    uint32_t key[VPT];
    #pragma unroll
    for (int v = 0; v < VPT; ++v) {
      x[v] = ahead[v];
      key[v] = live && lane + v * LPR < experts ? order_key(x[v]) : 0u;
    }
    if (VPT <= 8) fetch(row + kRows);
    float top = -INFINITY, mine = -INFINITY;
    int id = -1;
    for (int j = 0; j < k; ++j) {
      uint32_t best = 0;
      int at = 0;
      #pragma unroll
      for (int v = 0; v < VPT; ++v)
        if (v == 0 || key[v] > best) { best = key[v]; at = lane + v * LPR; }
      if (LPR == 32) {
        const uint32_t most = __reduce_max_sync(0xFFFFFFFFu, best);
        at = int(__reduce_min_sync(0xFFFFFFFFu, best == most ? uint32_t(at) : 0xFFFFFFFFu));
        best = most;
      } else {
        #pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) {
          const uint32_t ob = __shfl_xor_sync(0xFFFFFFFFu, best, o);
          const int oa = __shfl_xor_sync(0xFFFFFFFFu, at, o);
          if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
        }
      }
      const bool allowed = best > kKeyNone;
      if (j == 0 && allowed) top = key_value(best);
      if (lane == j && allowed) { mine = key_value(best); id = at; }
      #pragma unroll
      for (int v = 0; v < VPT; ++v)
        if (lane + v * LPR == at) key[v] = 0u;
    }
    const float m = top == -INFINITY ? 0.f : top;
    const float num = id >= 0 ? expf(mine - m) : 0.f;
    float sum = 0.f;
    if (normalize) {
      sum = num;
    } else {
      #pragma unroll
      for (int v = 0; v < VPT; ++v) sum += expf(x[v] - m);
    }
    #pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (live && lane < k) {
      weights[int64_t(row) * k + lane] = id >= 0 ? num / sum : 0.f;
      ids[int64_t(row) * k + lane] = id;
      atomicAdd(&hist[id >= 0 ? id : experts], 1);
    }
    if (VPT > 8) fetch(row + kRows);
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) counts[int64_t(blockIdx.x) * (experts + 1) + e] = hist[e];
}

// d logit_e = sum_j w_j (1[e = id_j] - p_e) dw_j, p the softmax the weights came from. One
// warp per row. The softmax over all experts needs no sums again: choice 0 is the largest
// logit, so p_e = w_0 exp(l_e - l_{id_0}).
template <typename T>
__global__ void __launch_bounds__(kBwdThreads) route_bwd_kernel(const T* __restrict__ logits, int64_t ld,
                                                                const float* __restrict__ weights,
                                                                const int* __restrict__ ids,
                                                                const float* __restrict__ dweights,
                                                                T* __restrict__ dlogits, int tokens, int experts,
                                                                int k, bool normalize) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * (kBwdThreads / 32) + (threadIdx.x >> 5);
  if (row >= tokens) return;
  int id = -1;
  float w = 0.f, dw = 0.f;
  if (lane < k) {
    id = ids[int64_t(row) * k + lane];
    w = weights[int64_t(row) * k + lane];
    dw = dweights[int64_t(row) * k + lane];
    if (id < 0) dw = 0.f;  // whatever arrives at a choice that was not made
  }
  float dot = w * dw;
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
  const float up = normalize ? w * (dw - dot) : w * dw;
  const T* x = logits + int64_t(row) * ld;
  const int id0 = __shfl_sync(0xFFFFFFFFu, id, 0);
  const float w0 = __shfl_sync(0xFFFFFFFFu, w, 0);
  const bool rest = !normalize && id0 >= 0 && id0 < experts;
  const float x0 = rest ? logit_at(x + id0) : 0.f;
  for (int e0 = 0; e0 < experts; e0 += 128) {  // four experts per lane
    float g[4];
    #pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int e = e0 + v * 32 + lane;
      g[v] = rest && e < experts ? -(w0 * expf(logit_at(x + e) - x0)) * dot : 0.f;
    }
    for (int j = 0; j < k; ++j) {
      const int ej = __shfl_sync(0xFFFFFFFFu, id, j);
      const float uj = __shfl_sync(0xFFFFFFFFu, up, j);
      #pragma unroll
      for (int v = 0; v < 4; ++v)
        if (e0 + v * 32 + lane == ej) g[v] += uj;
    }
    #pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int e = e0 + v * 32 + lane;
      if (e < experts) store_logit(dlogits + int64_t(row) * experts + e, g[v]);
    }
  }
}

// ---- plan -----------------------------------------------------------------------------

// Expert of pair i in 0..experts-1, or ``experts`` for a pair that no expert here takes.
__device__ __forceinline__ int expert_of(const int* __restrict__ ids, int64_t i, int start, int experts) {
  const int64_t e = int64_t(ids[i]) - start;
  return e >= 0 && e < experts ? int(e) : experts;
}

__global__ void __launch_bounds__(1024) plan_count_kernel(const int* __restrict__ ids, int64_t pairs,
                                                          int64_t pairs_per_block, int start, int experts,
                                                          int* __restrict__ counts) {
  pdl_enter();
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  const int64_t first = blockIdx.x * pairs_per_block, last = min(pairs, first + pairs_per_block);
  for (int64_t i = first + threadIdx.x; i < last; i += blockDim.x)
    atomicAdd(&hist[expert_of(ids, i, start, experts)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) counts[int64_t(blockIdx.x) * (experts + 1) + e] = hist[e];
}

// Shared memory: place[experts + 1] (next place of each expert for this block) and
// next[warps][experts + 1] (the same for each warp's run of the block's pairs).
__global__ void __launch_bounds__(1024) plan_place_kernel(const int* __restrict__ ids, int64_t pairs,
                                                          int64_t pairs_per_block, int start, int experts,
                                                          const int* __restrict__ counts,
                                                          int* __restrict__ offsets, int* __restrict__ slots) {
  pdl_enter();
  extern __shared__ int sm[];
  const int width = experts + 1;
  int* place = sm;
  int* total = sm + width;
  int* next = sm + 2 * width;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  for (int e = threadIdx.x; e < (2 + warps) * width; e += blockDim.x) sm[e] = 0;
  __syncthreads();
  // this block's pairs, one contiguous run per warp
  const int64_t first = blockIdx.x * pairs_per_block, last = min(pairs, first + pairs_per_block);
  const int64_t per_warp = ((pairs_per_block + warps - 1) / warps + 31) / 32 * 32;
  const int64_t wfirst = first + warp * per_warp, wlast = min(last, wfirst + per_warp);
  for (int64_t i = wfirst + lane; i < wlast; i += 32) atomicAdd(&next[warp * width + expert_of(ids, i, start, experts)], 1);
  const int cells = int(gridDim.x) * width;
  constexpr int kBatch = 8;  // loads under way per thread: the counts come from L2
  for (int c0 = threadIdx.x; c0 < cells; c0 += kBatch * blockDim.x) {
    int v[kBatch];
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) v[i] = c0 + i * int(blockDim.x) < cells ? counts[c0 + i * blockDim.x] : 0;
    #pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (v[i] == 0) continue;
      const int c = c0 + i * int(blockDim.x);
      const int b = c / width, e = c - b * width;
      atomicAdd(&total[e], v[i]);
      if (b < int(blockIdx.x)) atomicAdd(&place[e], v[i]);
    }
  }
  __syncthreads();
  // exclusive sum of the totals over the experts, by one warp
  if (warp == 0) {
    int carry = 0;
    for (int e0 = 0; e0 < width; e0 += 32) {
      const int e = e0 + lane;
      const int v = e < width ? total[e] : 0;
      int s = v;
      #pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, s, o);
        if (lane >= o) s += u;
      }
      if (e < width) total[e] = carry + s - v;
      carry += __shfl_sync(0xFFFFFFFFu, s, 31);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < width; e += blockDim.x) {
    if (blockIdx.x == 0) offsets[e] = total[e];
    int at = place[e] + total[e];
    for (int w = 0; w < warps; ++w) {
      const int n = next[w * width + e];
      next[w * width + e] = at;
      at += n;
    }
  }
  __syncthreads();
  int* mine = next + warp * width;
  for (int64_t i0 = wfirst; i0 < wlast; i0 += 32) {
    const int64_t i = i0 + lane;
    const int e = i < wlast ? expert_of(ids, i, start, experts) : -1;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    const int at = e >= 0 ? mine[e] : 0;
    __syncwarp();
    if (e >= 0) {
      slots[i] = at + before;
      if (before == 0) mine[e] = at + __popc(same);
    }
    __syncwarp();
  }
}

// ---- row movements --------------------------------------------------------------------

template <int VEC>
struct Row;
template <>
struct Row<8> {
  using Raw = uint4;
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[8]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __bfloat1622float2(h[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ Raw pack(const float (&f)[8]) {
    return make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
  }
  static __device__ __forceinline__ Raw zero() { return make_uint4(0, 0, 0, 0); }
};
template <>
struct Row<1> {
  using Raw = __nv_bfloat16;
  static __device__ __forceinline__ void unpack(const Raw& r, float (&f)[1]) { f[0] = __bfloat162float(r); }
  static __device__ __forceinline__ Raw pack(const float (&f)[1]) { return __float2bfloat16(f[0]); }
  static __device__ __forceinline__ Raw zero() { return __float2bfloat16(0.f); }
};

struct MoveArgs {
  const void* in;        // scatter: x / dout [tokens, d]; gather: y [rows, d]
  const void* y;         // scatter: the rows whose product with dout is dweights, or nullptr
  const float* weights;  // [tokens, k] or nullptr (ones)
  const void* residual;  // gather: [tokens, d] or nullptr
  void* out;
  float* dweights;
  const int* slots;
  const int* used;       // &offsets[experts]: places from here on hold nothing
  int tokens, k, d;
  int* err;
};

// The place of pair (t, j): -1 if it lies outside the rows (recorded), and whether an
// expert takes it.
__device__ __forceinline__ int place_of(const MoveArgs& a, int64_t pair, int used, bool& kept) {
  const int s = a.slots[pair];
  const bool ok = s >= 0 && int64_t(s) < int64_t(a.tokens) * a.k;
  if (!ok) record_error(a.err, kErrBounds);
  kept = ok && s < used;
  return ok ? s : -1;
}

// Choices handled together where few rows keep the SMs waiting: their places, then their rows,
// are asked for before the first is used (37 tokens of eight choices, width 5120: 3.3 us, one
// by one 4.0).
constexpr int kTogether = 4;

// Threads of a block: ``lpr`` per row (blockDim.x / lpr rows), grid.y over the row's vectors, U
// vectors per thread.
template <int VEC, int U, int J>
__global__ void __launch_bounds__(256) gather_kernel(MoveArgs a, int lpr) {
  pdl_enter();
  using R = Row<VEC>;
  using Raw = typename R::Raw;
  const int t = blockIdx.x * (blockDim.x / lpr) + threadIdx.x / lpr;
  const int v = blockIdx.y * lpr * U + threadIdx.x % lpr;
  const int vpr = a.d / VEC;
  if (t >= a.tokens || v >= vpr) return;
  const int used = *a.used;
  float acc[U][VEC];
  #pragma unroll
  for (int u = 0; u < U; ++u) {
    #pragma unroll
    for (int e = 0; e < VEC; ++e) acc[u][e] = 0.f;
    if (a.residual != nullptr && v + u * lpr < vpr)
      R::unpack(static_cast<const Raw*>(a.residual)[int64_t(t) * vpr + v + u * lpr], acc[u]);
  }
  for (int j0 = 0; j0 < a.k; j0 += J) {
    Raw raw[J][U];
    float w[J];
    bool kept[J];
    int s[J];
    #pragma unroll
    for (int j = 0; j < J; ++j) {
      const int64_t pair = int64_t(t) * a.k + j0 + j;
      kept[j] = false;
      if (j0 + j < a.k) s[j] = place_of(a, pair, used, kept[j]);
      w[j] = kept[j] && a.weights != nullptr ? a.weights[pair] : 1.f;
    }
    #pragma unroll
    for (int j = 0; j < J; ++j)
      #pragma unroll
      for (int u = 0; u < U; ++u)
        if (kept[j] && v + u * lpr < vpr) raw[j][u] = static_cast<const Raw*>(a.in)[int64_t(s[j]) * vpr + v + u * lpr];
    #pragma unroll
    for (int j = 0; j < J; ++j) {
      if (!kept[j]) continue;
      #pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v + u * lpr >= vpr) break;
        float f[VEC];
        R::unpack(raw[j][u], f);
        #pragma unroll
        for (int e = 0; e < VEC; ++e) acc[u][e] += w[j] * f[e];
      }
    }
  }
  #pragma unroll
  for (int u = 0; u < U; ++u)
    if (v + u * lpr < vpr) static_cast<Raw*>(a.out)[int64_t(t) * vpr + v + u * lpr] = R::pack(acc[u]);
}

// The same with a warp per token, U vectors per lane and J choices under way at a time; the
// warp's lanes fetch the token's places and weights together and hand them round. Many rows of
// at least 32 vectors: no block-wide step and no idle lane between a token's loads. 4096 tokens
// of two choices, width 2048, with residual: 11.4 us (5.9 TB/s) with U = J = 2; U = 4 12.5,
// J = 4 16.5 (fewer warps), a thread per vector 13.1.
template <int VEC, int U, int J>
__global__ void __launch_bounds__(256) gather_warp_kernel(MoveArgs a) {
  pdl_enter();
  using R = Row<VEC>;
  using Raw = typename R::Raw;
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int vpr = a.d / VEC;
  if (t >= a.tokens) return;
  const int used = *a.used;
  int place = -1;
  float weight = 0.f;
  if (lane < a.k) {
    bool kept;
    const int s = place_of(a, int64_t(t) * a.k + lane, used, kept);
    if (kept) {
      place = s;
      weight = a.weights != nullptr ? a.weights[int64_t(t) * a.k + lane] : 1.f;
    }
  }
  const Raw* res = static_cast<const Raw*>(a.residual) + int64_t(t) * vpr;
  Raw* out = static_cast<Raw*>(a.out) + int64_t(t) * vpr;
  for (int v0 = 0; v0 < vpr; v0 += 32 * U) {
    const int v = v0 + lane;
    float acc[U][VEC];
    #pragma unroll
    for (int u = 0; u < U; ++u) {
      #pragma unroll
      for (int e = 0; e < VEC; ++e) acc[u][e] = 0.f;
      if (a.residual != nullptr && v + u * 32 < vpr) R::unpack(res[v + u * 32], acc[u]);
    }
    for (int j0 = 0; j0 < a.k; j0 += J) {
      Raw raw[J][U];
      int s[J];
      float w[J];
      #pragma unroll
      for (int j = 0; j < J; ++j) {
        s[j] = __shfl_sync(0xFFFFFFFFu, place, (j0 + j) & 31);  // lanes from k on hold none
        w[j] = __shfl_sync(0xFFFFFFFFu, weight, (j0 + j) & 31);
        #pragma unroll
        for (int u = 0; u < U; ++u)
          if (s[j] >= 0 && v + u * 32 < vpr) raw[j][u] = static_cast<const Raw*>(a.in)[int64_t(s[j]) * vpr + v + u * 32];
      }
      #pragma unroll
      for (int j = 0; j < J; ++j) {
        if (s[j] < 0) continue;
        #pragma unroll
        for (int u = 0; u < U; ++u) {
          if (v + u * 32 >= vpr) break;
          float f[VEC];
          R::unpack(raw[j][u], f);
          #pragma unroll
          for (int e = 0; e < VEC; ++e) acc[u][e] += w[j] * f[e];
        }
      }
    }
    #pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * 32 < vpr) out[v + u * 32] = R::pack(acc[u]);
  }
}

// Copies of a token's row at its pairs' places; zeros where no expert takes the pair.
template <int VEC, int U>
__global__ void __launch_bounds__(256) scatter_kernel(MoveArgs a, int lpr) {
  pdl_enter();
  using R = Row<VEC>;
  using Raw = typename R::Raw;
  const int t = blockIdx.x * (blockDim.x / lpr) + threadIdx.x / lpr;
  const int v = blockIdx.y * lpr * U + threadIdx.x % lpr;
  const int vpr = a.d / VEC;
  if (t >= a.tokens || v >= vpr) return;
  const int used = *a.used;
  Raw raw[U];
  #pragma unroll
  for (int u = 0; u < U; ++u)
    if (v + u * lpr < vpr) raw[u] = static_cast<const Raw*>(a.in)[int64_t(t) * vpr + v + u * lpr];
  for (int j = 0; j < a.k; ++j) {
    bool kept;
    const int s = place_of(a, int64_t(t) * a.k + j, used, kept);
    if (s < 0) continue;
    #pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * lpr < vpr) static_cast<Raw*>(a.out)[int64_t(s) * vpr + v + u * lpr] = kept ? raw[u] : R::zero();
  }
}

// Combine's gradient: dy[slots[t, j]] = w[t, j] dout[t] and dw[t, j] = <y[slots[t, j]], dout[t]>.
// ``lpr`` lanes per pair (t, j), U vectors per lane at a time: one warp where there are pairs
// enough to fill the SMs with warps, up to a block where there are few. A token's dout is read
// once per choice, from the caches after the first. 4096 tokens of two choices, width 2048: a
// warp per pair 13.7 us (6.1 TB/s; U = 2 14.6, U = 8 16.3), a block per pair 23.6, a block per
// token with two choices at a time 20.7. The products are summed lane, warp, pair in a fixed
// order.
template <int VEC, int U>
__global__ void __launch_bounds__(256) combine_bwd_kernel(MoveArgs a, int lpr) {
  pdl_enter();
  using R = Row<VEC>;
  using Raw = typename R::Raw;
  __shared__ float part[8];
  const int64_t pair = int64_t(blockIdx.x) * (256 / lpr) + threadIdx.x / lpr;
  const int lane = threadIdx.x % lpr;
  const bool live = pair < int64_t(a.tokens) * a.k;
  const int vpr = a.d / VEC;
  const int used = *a.used;
  bool kept = false;
  const int s = live ? place_of(a, pair, used, kept) : -1;
  float dot = 0.f;
  if (s >= 0) {
    const Raw* dout = static_cast<const Raw*>(a.in) + int64_t(uint32_t(pair) / uint32_t(a.k)) * vpr;
    const Raw* y = static_cast<const Raw*>(a.y) + int64_t(s) * vpr;
    Raw* dy = static_cast<Raw*>(a.out) + int64_t(s) * vpr;
    if (kept) {
      const float w = a.weights != nullptr ? a.weights[pair] : 1.f;
      for (int v0 = lane; v0 < vpr; v0 += U * lpr) {
        Raw gr[U], yr[U];
        #pragma unroll
        for (int u = 0; u < U; ++u)
          if (v0 + u * lpr < vpr) {
            gr[u] = dout[v0 + u * lpr];
            yr[u] = y[v0 + u * lpr];
          }
        #pragma unroll
        for (int u = 0; u < U; ++u) {
          if (v0 + u * lpr >= vpr) break;
          float g[VEC], f[VEC];
          R::unpack(gr[u], g);
          R::unpack(yr[u], f);
          #pragma unroll
          for (int e = 0; e < VEC; ++e) {
            dot += f[e] * g[e];
            g[e] *= w;
          }
          dy[v0 + u * lpr] = R::pack(g);
        }
      }
    } else {
      for (int v = lane; v < vpr; v += lpr) dy[v] = R::zero();
    }
  }
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
  if (lpr > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
    __syncthreads();
    dot = 0.f;
    if (lane == 0)
      for (int i = 0; i < lpr / 32; ++i) dot += part[(threadIdx.x >> 5) + i];
  }
  if (live && lane == 0) a.dweights[pair] = dot;
}

// ---- launches -------------------------------------------------------------------------

int up(int64_t a, int64_t b) { return int((a + b - 1) / b); }

// Lanes per row: the power of two that holds a row's vectors, from 8 to 256.
int lanes_for(int vpr) {
  int l = 8;
  while (l < vpr && l < 256) l <<= 1;
  return l;
}

bool vectors(const MoveArgs& a) {
  const uintptr_t al = reinterpret_cast<uintptr_t>(a.in) | reinterpret_cast<uintptr_t>(a.y) |
                       reinterpret_cast<uintptr_t>(a.residual) | reinterpret_cast<uintptr_t>(a.out);
  return a.d % 8 == 0 && al % 16 == 0;
}

void check_move(const MoveArgs& a) {
  RESIHP_CHECK(a.k >= 1 && a.d >= 1 && a.tokens >= 0, "moe rows: sizes must be positive");
  RESIHP_CHECK(int64_t(a.tokens) * a.k <= INT32_MAX, "moe rows: tokens * k passes 31 bits");
}

template <int VEC, int U>
void launch_rows(void (*kernel)(MoveArgs, int), const MoveArgs& a, cudaStream_t st) {
  const int vpr = a.d / VEC, lpr = lanes_for(up(vpr, U));
  const dim3 grid(up(a.tokens, 256 / lpr), up(vpr, lpr * U));
  RESIHP_CHECK(grid.y <= 65535, "moe rows: width too large");
  RESIHP_CUDA_CHECK(launch_pdl(kernel, grid, 256, 0, st, a, lpr));
}

void launch_place(const int* ids, int64_t pairs, int64_t per_block, int blocks, int start, int experts,
                  const int* counts, int* offsets, int* slots, cudaStream_t st) {
  // As many warps as their tables leave within 48 KB: 32 up to 360 experts, 9 at 1024.
  const int table = (experts + 1) * int(sizeof(int));
  const int warps = std::min(32, 49152 / table - 2);
  RESIHP_CUDA_CHECK(launch_pdl(plan_place_kernel, blocks, 32 * warps, (2 + warps) * table, st, ids, pairs, per_block,
                               start, experts, counts, offsets, slots));
}

// Blocks of the counting sort: at least 1024 pairs each, at most one per SM (every block
// reads every block's counts).
int plan_blocks(int64_t pairs, int num_sms) { return std::max(1, std::min(num_sms, up(pairs, 1024))); }

template <typename T, int LPR, int VPT>
void launch_route_as(const void* logits, int64_t ld, int tokens, int experts, int k, bool normalize, int rows_per_block,
                     int blocks, float* weights, int* ids, int* counts, cudaStream_t st) {
  RESIHP_CUDA_CHECK(launch_pdl(route_kernel<T, LPR, VPT>, blocks, kRouteThreads<VPT>, (experts + 1) * int(sizeof(int)), st,
                               static_cast<const T*>(logits), ld, tokens, experts, k, normalize, rows_per_block, weights,
                               ids, counts));
}

template <typename T>
void launch_route(const void* logits, int64_t ld, int tokens, int experts, int k, bool normalize, int rows_per_block,
                  int blocks, float* weights, int* ids, int* counts, cudaStream_t st) {
#define RESIHP_ROUTE(LPR, VPT) \
  launch_route_as<T, LPR, VPT>(logits, ld, tokens, experts, k, normalize, rows_per_block, blocks, weights, ids, counts, st)
  if (experts <= 8) RESIHP_ROUTE(8, 1);
  else if (experts <= 16) RESIHP_ROUTE(16, 1);
  else if (experts <= 32) RESIHP_ROUTE(32, 1);
  else if (experts <= 64) RESIHP_ROUTE(32, 2);
  else if (experts <= 128) RESIHP_ROUTE(32, 4);
  else if (experts <= 256) RESIHP_ROUTE(32, 8);
  else RESIHP_ROUTE(32, 32);
#undef RESIHP_ROUTE
}

}  // namespace

int moe_blocks(int64_t pairs, int num_sms) { return plan_blocks(pairs, num_sms); }

void moe_route(const void* logits, bool bf16, int64_t ld, int tokens, int experts, int k, bool normalize,
               float* weights, int* ids, int* counts, int* offsets, int* slots, int num_sms, cudaStream_t st) {
  RESIHP_CHECK(experts >= 1 && experts <= kMoeMaxExperts, "moe_route takes 1 to ", kMoeMaxExperts, " experts");
  RESIHP_CHECK(k >= 1 && k <= kMoeMaxChoices && k <= experts, "moe_route takes 1 to ", kMoeMaxChoices,
               " choices, no more than experts");
  RESIHP_CHECK(int64_t(tokens) * k <= INT32_MAX, "moe_route: tokens * k passes 31 bits");
  const int64_t pairs = int64_t(tokens) * k;
  const int rows_per_block = std::max(1, up(tokens, plan_blocks(pairs, num_sms)));
  const int blocks = std::max(1, up(tokens, rows_per_block));
  if (bf16) launch_route<__nv_bfloat16>(logits, ld, tokens, experts, k, normalize, rows_per_block, blocks, weights, ids, counts, st);
  else launch_route<float>(logits, ld, tokens, experts, k, normalize, rows_per_block, blocks, weights, ids, counts, st);
  launch_place(ids, pairs, int64_t(rows_per_block) * k, blocks, 0, experts, counts, offsets, slots, st);
}

void moe_route_bwd(const void* logits, bool bf16, int64_t ld, const float* weights, const int* ids,
                   const float* dweights, void* dlogits, int tokens, int experts, int k, bool normalize,
                   cudaStream_t st) {
  if (tokens == 0) return;
  const int grid = up(tokens, kBwdThreads / 32);
  if (bf16)
    RESIHP_CUDA_CHECK(launch_pdl(route_bwd_kernel<__nv_bfloat16>, grid, kBwdThreads, 0, st,
                                 static_cast<const __nv_bfloat16*>(logits), ld, weights, ids, dweights,
                                 static_cast<__nv_bfloat16*>(dlogits), tokens, experts, k, normalize));
  else
    RESIHP_CUDA_CHECK(launch_pdl(route_bwd_kernel<float>, grid, kBwdThreads, 0, st, static_cast<const float*>(logits),
                                 ld, weights, ids, dweights, static_cast<float*>(dlogits), tokens, experts, k, normalize));
}

void moe_plan(const int* ids, int64_t pairs, int start, int experts, int* counts, int* offsets, int* slots, int num_sms,
              cudaStream_t st) {
  RESIHP_CHECK(experts >= 1 && experts <= kMoeMaxExperts, "moe_plan takes 1 to ", kMoeMaxExperts, " experts");
  RESIHP_CHECK(pairs <= INT32_MAX, "moe_plan: tokens * k passes 31 bits");
  const int64_t per_block = std::max(1, up(pairs, plan_blocks(pairs, num_sms)));
  const int blocks = std::max(1, up(pairs, per_block));
  RESIHP_CUDA_CHECK(launch_pdl(plan_count_kernel, blocks, 1024, (experts + 1) * int(sizeof(int)), st, ids, pairs,
                               per_block, start, experts, counts));
  launch_place(ids, pairs, per_block, blocks, start, experts, counts, offsets, slots, st);
}

void moe_scatter(const void* x, const int* slots, const int* used, void* out, int tokens, int k, int d, int* err,
                 cudaStream_t st) {
  MoveArgs a{x, nullptr, nullptr, nullptr, out, nullptr, slots, used, tokens, k, d, err};
  check_move(a);
  if (tokens == 0) return;
  if (vectors(a)) launch_rows<8, 1>(scatter_kernel<8, 1>, a, st);
  else launch_rows<1, 4>(scatter_kernel<1, 4>, a, st);
}

void moe_gather(const void* y, const float* weights, const void* residual, const int* slots, const int* used, void* out,
                int tokens, int k, int d, int* err, int num_sms, cudaStream_t st) {
  MoveArgs a{y, nullptr, weights, residual, out, nullptr, slots, used, tokens, k, d, err};
  check_move(a);
  if (tokens == 0) return;
  const bool many = tokens >= num_sms * 16;
  if (!vectors(a)) {
    launch_rows<1, 4>(gather_kernel<1, 4, kTogether>, a, st);
  } else if (many && d >= 256) {
    RESIHP_CUDA_CHECK(launch_pdl(gather_warp_kernel<8, 2, 2>, up(tokens, 8), 256, 0, st, a));
  } else {
    launch_rows<8, 1>(many ? gather_kernel<8, 1, 1> : gather_kernel<8, 1, kTogether>, a, st);
  }
}

void moe_combine_bwd(const void* dout, const void* y, const float* weights, const int* slots, const int* used, void* dy,
                     float* dweights, int tokens, int k, int d, int* err, int num_sms, cudaStream_t st) {
  MoveArgs a{dout, y, weights, nullptr, dy, dweights, slots, used, tokens, k, d, err};
  check_move(a);
  if (tokens == 0) return;
  const bool vec = vectors(a);
  const int vpr = vec ? d / 8 : d;
  const int lpr = int64_t(tokens) * k >= int64_t(num_sms) * 16 ? 32 : std::max(32, lanes_for(vpr));
  const int grid = up(int64_t(tokens) * k, 256 / lpr);
  auto kernel = vec ? (vpr <= lpr ? combine_bwd_kernel<8, 1> : combine_bwd_kernel<8, 4>) : combine_bwd_kernel<1, 4>;
  RESIHP_CUDA_CHECK(launch_pdl(kernel, grid, 256, 0, st, a, lpr));
}

}  // namespace resihp
