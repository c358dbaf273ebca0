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

constexpr int kRouteThreads = 256;
constexpr int kPlanThreads = 256;
constexpr int kPlanWarps = kPlanThreads / 32;

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

// LPR lanes share a row, lane l holds the logits l, l + LPR, ... Choice j ends up on lane j.
template <typename T, int LPR, int VPT>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(const T* __restrict__ logits, int64_t ld, int tokens,
                                                              int experts, int k, bool normalize, int rows_per_block,
                                                              float* __restrict__ weights, int* __restrict__ ids,
                                                              int* __restrict__ counts) {
  pdl_enter();
  extern __shared__ int hist[];  // [experts + 1]
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  constexpr int kRows = kRouteThreads / LPR;
  const int sub = threadIdx.x / LPR, lane = threadIdx.x % LPR;
  const int first = blockIdx.x * rows_per_block;
  const int last = min(tokens, first + rows_per_block);
  // whole warps walk together (the shuffles need every lane); rows past the end are idle
  for (int base = first; base < last; base += kRows) {
    const int row = base + sub;
    const bool live = row < last;
    float x[VPT];
    uint32_t key[VPT];
    #pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int e = lane + v * LPR;
      const bool in = live && e < experts;
      x[v] = in ? logit_at(logits + int64_t(row) * ld + e) : -INFINITY;
      key[v] = in ? order_key(x[v]) : 0u;
    }
    float mine = -INFINITY, top = -INFINITY;
    int id = -1;
    for (int j = 0; j < k; ++j) {
      uint64_t best = 0;  // (key, lowest index first)
      float bx = -INFINITY;
      #pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const uint64_t c = (uint64_t(key[v]) << 32) | uint32_t(~(lane + v * LPR));
        if (c > best) { best = c; bx = x[v]; }
      }
      #pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) {
        const uint64_t c = __shfl_xor_sync(0xFFFFFFFFu, best, o);
        const float cx = __shfl_xor_sync(0xFFFFFFFFu, bx, o);
        if (c > best) { best = c; bx = cx; }
      }
      const int e = int(~uint32_t(best));
      const bool allowed = uint32_t(best >> 32) > kKeyNone;
      if (j == 0 && allowed) top = bx;
      if (lane == j && allowed) { mine = bx; id = e; }
      #pragma unroll
      for (int v = 0; v < VPT; ++v)
        if (lane + v * LPR == e) key[v] = 0u;
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
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) counts[int64_t(blockIdx.x) * (experts + 1) + e] = hist[e];
}

// d logit_e = sum_j w_j (1[e = id_j] - p_e) dw_j, p the softmax the weights came from. One
// warp per row; the softmax over all experts is computed again from the logits.
template <typename T>
__global__ void __launch_bounds__(kRouteThreads) route_bwd_kernel(const T* __restrict__ logits, int64_t ld,
                                                                  const float* __restrict__ weights,
                                                                  const int* __restrict__ ids,
                                                                  const float* __restrict__ dweights,
                                                                  T* __restrict__ dlogits, int tokens, int experts,
                                                                  int k, bool normalize) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * (kRouteThreads / 32) + (threadIdx.x >> 5);
  if (row >= tokens) return;
  int id = -1;
  float w = 0.f, dw = 0.f;
  if (lane < k) {
    id = ids[int64_t(row) * k + lane];
    if (id >= 0) {
      w = weights[int64_t(row) * k + lane];
      dw = dweights[int64_t(row) * k + lane];
    }
  }
  float dot = w * dw;
  #pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
  const T* x = logits + int64_t(row) * ld;
  float m = -INFINITY, sum = 0.f;
  if (!normalize) {
    for (int e = lane; e < experts; e += 32) m = fmaxf(m, logit_at(x + e));
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if (m == -INFINITY) m = 0.f;
    for (int e = lane; e < experts; e += 32) sum += expf(logit_at(x + e) - m);
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int e = e0 + lane;
    float g = 0.f;
    if (!normalize && e < experts) g = -(expf(logit_at(x + e) - m) * inv) * dot;
    for (int j = 0; j < k; ++j) {
      const int ej = __shfl_sync(0xFFFFFFFFu, id, j);
      const float wj = __shfl_sync(0xFFFFFFFFu, w, j), dj = __shfl_sync(0xFFFFFFFFu, dw, j);
      if (ej == e && ej >= 0) g += normalize ? wj * (dj - dot) : wj * dj;
    }
    if (e < experts) store_logit(dlogits + int64_t(row) * experts + e, g);
  }
}

// ---- plan -----------------------------------------------------------------------------

// Expert of pair i in 0..experts-1, or ``experts`` for a pair that no expert here takes.
__device__ __forceinline__ int expert_of(const int* __restrict__ ids, int64_t i, int start, int experts) {
  const int64_t e = int64_t(ids[i]) - start;
  return e >= 0 && e < experts ? int(e) : experts;
}

__global__ void __launch_bounds__(kPlanThreads) plan_count_kernel(const int* __restrict__ ids, int64_t pairs,
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
__global__ void __launch_bounds__(kPlanThreads) plan_place_kernel(const int* __restrict__ ids, int64_t pairs,
                                                                  int64_t pairs_per_block, int start, int experts,
                                                                  const int* __restrict__ counts,
                                                                  int* __restrict__ offsets, int* __restrict__ slots) {
  pdl_enter();
  extern __shared__ int sm[];
  const int width = experts + 1;
  int* place = sm;
  int* total = sm + width;
  int* next = sm + 2 * width;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < (2 + kPlanWarps) * width; e += blockDim.x) sm[e] = 0;
  __syncthreads();
  // this block's pairs, one contiguous run per warp
  const int64_t first = blockIdx.x * pairs_per_block, last = min(pairs, first + pairs_per_block);
  const int64_t per_warp = ((pairs_per_block + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
  const int64_t wfirst = first + warp * per_warp, wlast = min(last, wfirst + per_warp);
  for (int64_t i = wfirst + lane; i < wlast; i += 32) atomicAdd(&next[warp * width + expert_of(ids, i, start, experts)], 1);
  const int cells = int(gridDim.x) * width;
  for (int c = threadIdx.x; c < cells; c += blockDim.x) {
    const int v = counts[c];
    if (v == 0) continue;
    const int b = c / width, e = c - b * width;
    atomicAdd(&total[e], v);
    if (b < int(blockIdx.x)) atomicAdd(&place[e], v);
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
    for (int w = 0; w < kPlanWarps; ++w) {
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

// Threads of a block: ``lpr`` per row (blockDim.x / lpr rows), grid.y over the row's vectors.
template <int VEC>
__global__ void __launch_bounds__(256) gather_kernel(MoveArgs a, int lpr) {
  pdl_enter();
  using R = Row<VEC>;
  using Raw = typename R::Raw;
  const int t = blockIdx.x * (blockDim.x / lpr) + threadIdx.x / lpr;
  const int v = blockIdx.y * lpr + threadIdx.x % lpr;
  const int vpr = a.d / VEC;
  if (t >= a.tokens || v >= vpr) return;
  const int used = *a.used;
  float acc[VEC];
  #pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  if (a.residual != nullptr) R::unpack(static_cast<const Raw*>(a.residual)[int64_t(t) * vpr + v], acc);
  for (int j = 0; j < a.k; ++j) {
    const int64_t pair = int64_t(t) * a.k + j;
    bool kept;
    const int s = place_of(a, pair, used, kept);
    if (!kept) continue;
    float f[VEC];
    R::unpack(static_cast<const Raw*>(a.in)[int64_t(s) * vpr + v], f);
    const float w = a.weights != nullptr ? a.weights[pair] : 1.f;
    #pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] += w * f[e];
  }
  static_cast<Raw*>(a.out)[int64_t(t) * vpr + v] = R::pack(acc);
}

// Copies of a token's row (times its weights) at its pairs' places; zeros where no expert
// takes the pair.
template <int VEC>
__global__ void __launch_bounds__(256) scatter_kernel(MoveArgs a, int lpr) {
  pdl_enter();
  using R = Row<VEC>;
  using Raw = typename R::Raw;
  const int t = blockIdx.x * (blockDim.x / lpr) + threadIdx.x / lpr;
  const int v = blockIdx.y * lpr + threadIdx.x % lpr;
  const int vpr = a.d / VEC;
  if (t >= a.tokens || v >= vpr) return;
  const int used = *a.used;
  const Raw raw = static_cast<const Raw*>(a.in)[int64_t(t) * vpr + v];
  for (int j = 0; j < a.k; ++j) {
    bool kept;
    const int s = place_of(a, int64_t(t) * a.k + j, used, kept);
    if (s >= 0) static_cast<Raw*>(a.out)[int64_t(s) * vpr + v] = kept ? raw : R::zero();
  }
}

// Combine's gradient: dy[slots[t, j]] = w[t, j] dout[t] and dw[t, j] = <y[slots[t, j]], dout[t]>.
// One block per token; the products are summed lane, warp, block in a fixed order.
template <int VEC>
__global__ void __launch_bounds__(256) combine_bwd_kernel(MoveArgs a) {
  pdl_enter();
  using R = Row<VEC>;
  using Raw = typename R::Raw;
  __shared__ float part[8];
  const int t = blockIdx.x;
  const int vpr = a.d / VEC;
  const int used = *a.used;
  const Raw* dout = static_cast<const Raw*>(a.in) + int64_t(t) * vpr;
  for (int j = 0; j < a.k; ++j) {
    const int64_t pair = int64_t(t) * a.k + j;
    bool kept;
    const int s = place_of(a, pair, used, kept);
    const float w = a.weights != nullptr ? a.weights[pair] : 1.f;
    float dot = 0.f;
    if (s >= 0) {
      Raw* dy = static_cast<Raw*>(a.out) + int64_t(s) * vpr;
      const Raw* y = static_cast<const Raw*>(a.y) + int64_t(s) * vpr;
      for (int v = threadIdx.x; v < vpr; v += blockDim.x) {
        if (!kept) {
          dy[v] = R::zero();
          continue;
        }
        float g[VEC], f[VEC];
        R::unpack(dout[v], g);
        R::unpack(y[v], f);
        #pragma unroll
        for (int e = 0; e < VEC; ++e) {
          dot += f[e] * g[e];
          g[e] *= w;
        }
        dy[v] = R::pack(g);
      }
    }
    #pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
      float sum = 0.f;
      for (int w2 = 0; w2 < int(blockDim.x >> 5); ++w2) sum += part[w2];
      a.dweights[pair] = sum;
    }
    __syncthreads();
  }
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

template <int VEC>
void launch_rows(void (*kernel)(MoveArgs, int), const MoveArgs& a, cudaStream_t st) {
  const int vpr = a.d / VEC, lpr = lanes_for(vpr);
  const dim3 grid(up(a.tokens, 256 / lpr), up(vpr, lpr));
  RESIHP_CHECK(grid.y <= 65535, "moe rows: width too large");
  RESIHP_CUDA_CHECK(launch_pdl(kernel, grid, 256, 0, st, a, lpr));
}

void launch_place(const int* ids, int64_t pairs, int64_t per_block, int blocks, int start, int experts,
                  const int* counts, int* offsets, int* slots, cudaStream_t st) {
  const int smem = (2 + kPlanWarps) * (experts + 1) * int(sizeof(int));
  RESIHP_CUDA_CHECK(launch_pdl(plan_place_kernel, blocks, kPlanThreads, smem, st, ids, pairs, per_block, start, experts,
                               counts, offsets, slots));
}

// Blocks of the counting sort: at least 1024 pairs each, at most one per SM (every block
// reads every block's counts).
int plan_blocks(int64_t pairs, int num_sms) { return std::max(1, std::min(num_sms, up(pairs, 1024))); }

template <typename T, int LPR, int VPT>
void launch_route_as(const void* logits, int64_t ld, int tokens, int experts, int k, bool normalize, int rows_per_block,
                     int blocks, float* weights, int* ids, int* counts, cudaStream_t st) {
  RESIHP_CUDA_CHECK(launch_pdl(route_kernel<T, LPR, VPT>, blocks, kRouteThreads, (experts + 1) * int(sizeof(int)), st,
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
  const int grid = up(tokens, kRouteThreads / 32);
  if (bf16)
    RESIHP_CUDA_CHECK(launch_pdl(route_bwd_kernel<__nv_bfloat16>, grid, kRouteThreads, 0, st,
                                 static_cast<const __nv_bfloat16*>(logits), ld, weights, ids, dweights,
                                 static_cast<__nv_bfloat16*>(dlogits), tokens, experts, k, normalize));
  else
    RESIHP_CUDA_CHECK(launch_pdl(route_bwd_kernel<float>, grid, kRouteThreads, 0, st, static_cast<const float*>(logits),
                                 ld, weights, ids, dweights, static_cast<float*>(dlogits), tokens, experts, k, normalize));
}

void moe_plan(const int* ids, int64_t pairs, int start, int experts, int* counts, int* offsets, int* slots, int num_sms,
              cudaStream_t st) {
  RESIHP_CHECK(experts >= 1 && experts <= kMoeMaxExperts, "moe_plan takes 1 to ", kMoeMaxExperts, " experts");
  RESIHP_CHECK(pairs <= INT32_MAX, "moe_plan: tokens * k passes 31 bits");
  const int64_t per_block = std::max(1, up(pairs, plan_blocks(pairs, num_sms)));
  const int blocks = std::max(1, up(pairs, per_block));
  RESIHP_CUDA_CHECK(launch_pdl(plan_count_kernel, blocks, kPlanThreads, (experts + 1) * int(sizeof(int)), st, ids, pairs,
                               per_block, start, experts, counts));
  launch_place(ids, pairs, per_block, blocks, start, experts, counts, offsets, slots, st);
}

void moe_scatter(const void* x, const int* slots, const int* used, void* out, int tokens, int k, int d, int* err,
                 cudaStream_t st) {
  MoveArgs a{x, nullptr, nullptr, nullptr, out, nullptr, slots, used, tokens, k, d, err};
  check_move(a);
  if (tokens == 0) return;
  if (vectors(a)) launch_rows<8>(scatter_kernel<8>, a, st);
  else launch_rows<1>(scatter_kernel<1>, a, st);
}

void moe_gather(const void* y, const float* weights, const void* residual, const int* slots, const int* used, void* out,
                int tokens, int k, int d, int* err, cudaStream_t st) {
  MoveArgs a{y, nullptr, weights, residual, out, nullptr, slots, used, tokens, k, d, err};
  check_move(a);
  if (tokens == 0) return;
  if (vectors(a)) launch_rows<8>(gather_kernel<8>, a, st);
  else launch_rows<1>(gather_kernel<1>, a, st);
}

void moe_combine_bwd(const void* dout, const void* y, const float* weights, const int* slots, const int* used, void* dy,
                     float* dweights, int tokens, int k, int d, int* err, cudaStream_t st) {
  MoveArgs a{dout, y, weights, nullptr, dy, dweights, slots, used, tokens, k, d, err};
  check_move(a);
  if (tokens == 0) return;
  const bool vec = vectors(a);
  const int vpr = vec ? d / 8 : d;
  const int block = std::min(256, up(vpr, 32) * 32);
  RESIHP_CUDA_CHECK(launch_pdl(vec ? combine_bwd_kernel<8> : combine_bwd_kernel<1>, tokens, block, 0, st, a));
}

}  // namespace resihp
