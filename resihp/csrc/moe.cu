// Routing of a sparse (mixture-of-experts) MLP around its per-expert products (no
// counterpart in the reference, whose blocks are dense): the router's choice of experts,
// the plan that sorts the (token, choice) pairs by expert, and the two row movements.
//
//   route     ids[t, j] = the expert of token t's j-th largest logit (lowest index first
//             among equal ones), weights = softmax over all experts or over the chosen ones
//   plan      offsets[e] = pairs of the experts before e;  slots[t, j] = the pair's place in
//             the order (expert, token, choice); pairs of no expert go behind offsets[E]
//   scatter   y[slots[t, j]] = x[t]                        (dispatch; combine's gradient
//             y[slots[t, j]] = w[t, j] x[t] goes with its dot products)
//   gather    out[t] = residual[t] + sum_j w[t, j] y[slots[t, j]]   (combine; dispatch's)
//
// The plan is a stable counting sort in two launches: the first counts experts per run of
// consecutive pairs, the second adds up the counts of the runs before its own, ranks its
// pairs warp by warp and writes their places. Nothing is decided by the order of atomics
// (they only count), so a plan is the same on every run; and no state outlives a call.
//
// The row movements go by token (or by pair, one token's pairs side by side), so a token's row
// comes from memory once however many experts it has. Per token k + 1 rows move in dispatch, its
// gradient and combine (k + 2 with a residual), 2 k + 1 in combine's gradient: no more than has
// to. They are bound by memory: 4096 tokens of two choices, width 2048, on rows that are not in
// L2, take 9.4 us for dispatch, 12.8 for combine with a residual, 9.9 and 15.3 for their gradients
// (5.1 to 5.5 TB/s of the 6.5 a copy reaches); with three sets of rows in turn, partly from L2,
// 7.2, 11.6, 8.6 and 13.5. Rows of an odd width have no common alignment and move two bytes at a
// time: 1021 tokens of six choices, width 1003, take 5.7 us out and 10.5 back, where their bytes
// take 2.2.
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace resihp {

namespace {

// ---- routing --------------------------------------------------------------------------

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

// ---- plan -----------------------------------------------------------------------------

// Expert of pair i in 0..experts-1, or ``experts`` for a pair that no expert here takes.
__device__ __forceinline__ int expert_of(const int* ids, int64_t i, int start, int experts) {
  const int64_t e = int64_t(ids[i]) - start;
  return e >= 0 && e < experts ? int(e) : experts;
}

__global__ void __launch_bounds__(1024) moe_plan_count_kernel(const int* __restrict__ ids, int64_t pairs,
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

// The places of the pairs first .. last - 1 (per_block of them in every block but the last), by
// one block. total[e]: all pairs of expert e; place[e]: those in the blocks before this one;
// next: [warps][experts + 1] scratch. All in shared memory. Each warp takes a run of consecutive
// pairs: it counts them, learns where its run starts within each expert, and hands out places
// 32 pairs at a time, equal experts in lane order.
__device__ __forceinline__ void place_pairs(const int* ids, int64_t first, int64_t last, int64_t per_block, int start,
                                            int experts, int* total, int* place, int* next, int* offsets, int* slots) {
  const int width = experts + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  for (int e = threadIdx.x; e < warps * width; e += blockDim.x) next[e] = 0;
  __syncthreads();
  const int64_t per_warp = ((per_block + warps - 1) / warps + 31) / 32 * 32;
  const int64_t wfirst = first + warp * per_warp, wlast = min(last, wfirst + per_warp);
  for (int64_t i = wfirst + lane; i < wlast; i += 32) atomicAdd(&next[warp * width + expert_of(ids, i, start, experts)], 1);
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

__global__ void __launch_bounds__(1024) moe_plan_place_kernel(const int* __restrict__ ids, int64_t pairs,
                                                          int64_t pairs_per_block, int start, int experts,
                                                          const int* __restrict__ counts,
                                                          int* __restrict__ offsets, int* __restrict__ slots) {
  pdl_enter();
  extern __shared__ int sm[];
  const int width = experts + 1, blocks = int(gridDim.x), me = int(blockIdx.x);
  int* total = sm;
  int* place = sm + width;
  for (int e = threadIdx.x; e < 2 * width; e += blockDim.x) sm[e] = 0;
  __syncthreads();
  // column sums of the blocks' counts: as many threads per expert as there are
  const int parts = max(1, int(blockDim.x) / width);
  for (int c = threadIdx.x; c < parts * width; c += blockDim.x) {
    const int part = c / width, e = c - part * width;
    int all = 0, before = 0;
    #pragma unroll 8
    for (int b = part; b < blocks; b += parts) {
      const int v = counts[int64_t(b) * width + e];
      all += v;
      if (b < me) before += v;
    }
    atomicAdd(&total[e], all);
    atomicAdd(&place[e], before);
  }
  const int64_t first = blockIdx.x * pairs_per_block;
  place_pairs(ids, first, min(pairs, first + pairs_per_block), pairs_per_block, start, experts, total, place,
              sm + 2 * width, offsets, slots);
}

// LPR lanes share a row, lane l holds the logits l, l + LPR, ...: eight to 32 per lane, so that
// most of a choice is found within lanes and a warp serves 32 / LPR rows (a warp per row with
// warp-wide reductions took 14 us for 32768 rows of 64 experts, four choices; this takes 9).
// Lane j % LPR keeps choice j. A grid of one block goes on to sort its pairs itself.
template <typename T, int LPR, int VPT, int KMAX>
__global__ void __launch_bounds__(512) moe_route_kernel(const T* __restrict__ logits, int64_t ld, int tokens, int experts,
                                                    int k, bool normalize, int rows_per_block,
                                                    float* __restrict__ weights, int* ids, int* __restrict__ counts,
                                                    int* __restrict__ offsets, int* __restrict__ slots) {
  pdl_enter();
  extern __shared__ int sm[];
  int* hist = sm;  // [experts + 1]
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  constexpr int kMine = (KMAX + LPR - 1) / LPR;  // choices a lane keeps: lane, lane + LPR, ...
  const int rows = blockDim.x / LPR;
  const int sub = threadIdx.x / LPR, lane = threadIdx.x % LPR;
  const int first = blockIdx.x * rows_per_block;
  const int last = min(tokens, first + rows_per_block);
  // whole warps walk together (the shuffles need every lane); rows past the end are idle
  for (int base = first; base < last; base += rows) {
    const int row = base + sub;
    const bool live = row < last;
    float x[VPT];
    uint32_t key[VPT];
    #pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int e = lane + v * LPR;
      x[v] = live && e < experts ? logit_at(logits + int64_t(row) * ld + e) : -INFINITY;
    }
    #pragma unroll
    for (int v = 0; v < VPT; ++v) key[v] = live && lane + v * LPR < experts ? order_key(x[v]) : 0u;
    float m = 0.f, mine[kMine];
    int id[kMine];
    #pragma unroll
    for (int i = 0; i < kMine; ++i) id[i] = -1;
    #pragma unroll 1
    for (int j = 0; j < k; ++j) {
      uint32_t best = key[0];
      int at = lane;
      #pragma unroll
      for (int v = 1; v < VPT; ++v)
        if (key[v] > best) { best = key[v]; at = lane + v * LPR; }
      #pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) {
        const uint32_t ob = __shfl_xor_sync(0xFFFFFFFFu, best, o);
        const int oa = __shfl_xor_sync(0xFFFFFFFFu, at, o);
        if (ob > best || (ob == best && oa < at)) { best = ob; at = oa; }
      }
      const bool allowed = best > kKeyNone;
      const float value = key_value(best);
      if (j == 0 && allowed) m = value;
      #pragma unroll
      for (int i = 0; i < kMine; ++i)
        if (lane + i * LPR == j && allowed) { mine[i] = value; id[i] = at; }
      #pragma unroll
      for (int v = 0; v < VPT; ++v)
        if (lane + v * LPR == at) key[v] = 0u;
    }
    float sum = 0.f;
    #pragma unroll
    for (int i = 0; i < kMine; ++i) {
      mine[i] = id[i] >= 0 ? expf(mine[i] - m) : 0.f;
      if (normalize) sum += mine[i];
    }
    if (!normalize) {
      #pragma unroll
      for (int v = 0; v < VPT; ++v) sum += expf(x[v] - m);
    }
    #pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    #pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const int j = lane + i * LPR;
      if (live && j < k) {
        weights[int64_t(row) * k + j] = id[i] >= 0 ? mine[i] / sum : 0.f;
        ids[int64_t(row) * k + j] = id[i];
        atomicAdd(&hist[id[i] >= 0 ? id[i] : experts], 1);
      }
    }
  }
  __syncthreads();
  if (gridDim.x > 1) {
    for (int e = threadIdx.x; e <= experts; e += blockDim.x)
      counts[int64_t(blockIdx.x) * (experts + 1) + e] = hist[e];
    return;
  }
  // one block: the totals are its own, and no pair comes before its first
  int* place = sm + experts + 1;
  for (int e = threadIdx.x; e <= experts; e += blockDim.x) place[e] = 0;
  place_pairs(ids, 0, int64_t(tokens) * k, int64_t(tokens) * k, 0, experts, hist, place, place + experts + 1, offsets,
              slots);
}

// d logit_e = sum_j w_j (1[e = id_j] - p_e) dw_j, p the softmax the weights came from. lpr lanes
// per row, eight experts each at a time; every lane reads the row's choices, so nothing passes
// between lanes. The softmax over all experts needs no sums again: choice 0 is the largest
// logit, so p_e = w_0 exp(l_e - l_{id_0}).
template <typename T, int KMAX>
__global__ void __launch_bounds__(256) moe_route_bwd_kernel(const T* __restrict__ logits, int64_t ld,
                                                        const float* __restrict__ weights, const int* __restrict__ ids,
                                                        const float* __restrict__ dweights, T* __restrict__ dlogits,
                                                        int tokens, int experts, int k, bool normalize, int lpr) {
  pdl_enter();
  constexpr int kEach = 8;
  const int row = blockIdx.x * (256 / lpr) + threadIdx.x / lpr;
  const int lane = threadIdx.x % lpr;
  if (row >= tokens) return;
  const T* x = logits + int64_t(row) * ld;
  float l[kEach];
  if (!normalize) {  // on their way while the choices arrive
    #pragma unroll
    for (int v = 0; v < kEach; ++v) l[v] = lane + v * lpr < experts ? logit_at(x + lane + v * lpr) : -INFINITY;
  }
  int id[KMAX];
  float up[KMAX];
  float dot = 0.f, w0 = 0.f;
  #pragma unroll
  for (int j = 0; j < KMAX; ++j) {
    id[j] = -1;
    up[j] = 0.f;
    if (j < k) {
      id[j] = ids[int64_t(row) * k + j];
      const float w = weights[int64_t(row) * k + j];
      if (j == 0) w0 = w;
      // whatever arrives at a choice that was not made counts for nothing
      if (id[j] >= 0) up[j] = w * dweights[int64_t(row) * k + j];
      dot += up[j];
    }
  }
  if (normalize) {
    #pragma unroll
    for (int j = 0; j < KMAX; ++j)
      if (j < k && id[j] >= 0) up[j] -= weights[int64_t(row) * k + j] * dot;
  }
  const bool rest = !normalize && id[0] >= 0 && id[0] < experts;
  const float x0 = rest ? logit_at(x + id[0]) : 0.f;
  for (int e0 = 0; e0 < experts; e0 += kEach * lpr) {
    #pragma unroll
    for (int v = 0; v < kEach; ++v) {
      const int e = e0 + lane + v * lpr;
      if (e >= experts) break;
      const float le = e0 == 0 || normalize ? l[v] : logit_at(x + e);
      float g = rest ? -(w0 * expf(le - x0)) * dot : 0.f;
      #pragma unroll
      for (int j = 0; j < KMAX; ++j)
        if (id[j] == e) g += up[j];
      store_logit(dlogits + int64_t(row) * experts + e, g);
    }
  }
}

// ---- row movements --------------------------------------------------------------------

// A row as 16-byte vectors, or element by element where its width or address forbids them.
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
  const float* weights;  // [tokens, k]; gather: or nullptr (ones)
  const void* residual;  // gather: [tokens, d] or nullptr
  void* out;
  float* dweights;
  const int* slots;
  const int* used;       // &offsets[experts]: places from here on hold nothing
  int tokens, k, d;
  int* err;
  int spans;  // scatter, combine's gradient: leading blocks that zero the rows without a pair
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

// Rows that no pair names, of the kSpan rows from ``span * kSpan`` on, become zeros: a plan made
// elsewhere may name a row twice or places out of range, and what lies in memory must not reach
// a weight gradient through the rows it leaves out. One block looks through all places, marks
// those of its rows and zeros the others; it depends on no other block, and where a plan is
// whole it writes nothing. It runs beside the blocks that move the rows, first of the grid. (Inline:
// behind a call the movers lose a tenth at odd widths. Marks are bytes: bits need atomics, twice
// the time.)
constexpr int kSpan = 16384;

template <int VEC>
__device__ __forceinline__ void zero_unnamed(const MoveArgs& a, int span) {
  using R = Row<VEC>;
  __shared__ __align__(16) uint8_t named[kSpan];
  const unsigned pairs = unsigned(a.tokens) * unsigned(a.k);  // (at most kMoeMaxPairs)
  const unsigned first = unsigned(span) * unsigned(kSpan);
  const unsigned rows = min(unsigned(kSpan), pairs - first);
  for (int i = threadIdx.x; i < kSpan / 16; i += 256) reinterpret_cast<uint4*>(named)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  auto mark = [&](int s) {
    const unsigned at = unsigned(s) - first;  // (negative places are far past ``rows``)
    if (at < rows) named[at] = 1;
  };
  // 16-byte loads between the first and last aligned ones, four under way per thread
  const unsigned lead = min(pairs, unsigned((4 - ((reinterpret_cast<uintptr_t>(a.slots) >> 2) & 3)) & 3));
  const unsigned quads = (pairs - lead) >> 2;
  const int4* body = reinterpret_cast<const int4*>(a.slots + lead);
  if (threadIdx.x < lead) mark(a.slots[threadIdx.x]);
  for (unsigned i0 = threadIdx.x; i0 < quads; i0 += 4 * 256) {
    int4 q[4];
    #pragma unroll
    for (int u = 0; u < 4; ++u) q[u] = i0 + u * 256 < quads ? body[i0 + u * 256] : make_int4(-1, -1, -1, -1);
    #pragma unroll
    for (int u = 0; u < 4; ++u) {
      mark(q[u].x);
      mark(q[u].y);
      mark(q[u].z);
      mark(q[u].w);
    }
  }
  for (unsigned i = lead + 4 * quads + threadIdx.x; i < pairs; i += 256) mark(a.slots[i]);
  __syncthreads();
  bool missing = false;
  for (unsigned i = threadIdx.x; i < rows / 4; i += 256) missing |= reinterpret_cast<const uint32_t*>(named)[i] != 0x01010101u;
  for (unsigned i = rows / 4 * 4 + threadIdx.x; i < rows; i += 256) missing |= named[i] == 0;
  if (!__syncthreads_or(missing)) return;
  const int vpr = a.d / VEC;
  for (unsigned r = threadIdx.x >> 5; r < rows; r += 8) {
    if (named[r]) continue;
    typename R::Raw* row = static_cast<typename R::Raw*>(a.out) + (int64_t(first) + r) * vpr;
    for (int v = threadIdx.x & 31; v < vpr; v += 32) row[v] = R::zero();
  }
}

// Choices handled together where few rows keep the SMs waiting: their places, then their rows,
// are asked for before the first is used (37 tokens of eight choices, width 5120: 3.3 us, one
// by one 4.0).
constexpr int kTogether = 4;

// Threads of a block: ``lpr`` per row (blockDim.x / lpr rows), grid.y over the row's vectors, U
// vectors per thread.
template <int VEC, int U, int J>
__global__ void __launch_bounds__(256) moe_gather_kernel(MoveArgs a, int lpr) {
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
// of two choices, width 2048, with residual (three sets in turn): 11.4 us with U = J = 2; U = 4
// 12.5, J = 4 16.5 (fewer warps), a thread per vector 13.1.
template <int VEC, int U, int J>
__global__ void __launch_bounds__(256) moe_gather_warp_kernel(MoveArgs a) {
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
        s[j] = __shfl_sync(0xFFFFFFFFu, place, j0 + j);  // lanes from k on hold none (k even or below 32)
        w[j] = __shfl_sync(0xFFFFFFFFu, weight, j0 + j);
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

// Copies of a token's row at its pairs' places; zeros where no expert takes the pair. (Registers
// for eight blocks per SM: with the 40 that zero_unnamed would take, 7.9 us instead of 7.4 for 4096
// tokens of two choices, width 2048.)
template <int VEC, int U>
__global__ void __launch_bounds__(256, 8) moe_scatter_kernel(MoveArgs a, int lpr) {
  pdl_enter();
  using R = Row<VEC>;
  using Raw = typename R::Raw;
  const int block = int(blockIdx.x) - a.spans;
  if (block < 0) {
    if (blockIdx.y == 0) zero_unnamed<VEC>(a, blockIdx.x);
    return;
  }
  const int t = block * (blockDim.x / lpr) + threadIdx.x / lpr;
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
// warp per pair 13.7 us (three sets in turn; U = 2 14.6, U = 8 16.3), a block per pair 23.6, a
// block per token with two choices at a time 20.7. The products are summed lane, warp, pair in a fixed
// order.
template <int VEC, int U>
__global__ void __launch_bounds__(256) moe_combine_bwd_kernel(MoveArgs a, int lpr) {
  pdl_enter();
  using R = Row<VEC>;
  using Raw = typename R::Raw;
  __shared__ float part[8];
  const int block = int(blockIdx.x) - a.spans;
  if (block < 0) {
    zero_unnamed<VEC>(a, blockIdx.x);
    return;
  }
  const int64_t pair = int64_t(block) * (256 / lpr) + threadIdx.x / lpr;
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
      const float w = a.weights[pair];
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
  RESIHP_CHECK(int64_t(a.tokens) * a.k <= kMoeMaxPairs, "moe rows: tokens * k passes ", kMoeMaxPairs);
}

template <int VEC, int U>
void launch_rows(void (*kernel)(MoveArgs, int), const MoveArgs& a, cudaStream_t st) {
  const int vpr = a.d / VEC, lpr = lanes_for(up(vpr, U));
  const dim3 grid(up(a.tokens, 256 / lpr) + a.spans, up(vpr, lpr * U));
  RESIHP_CHECK(grid.y <= 65535, "moe rows: width too large");
  RESIHP_CUDA_CHECK(launch_pdl(kernel, grid, 256, 0, st, a, lpr));
}

// The rows without a pair: blocks of zero_unnamed (``a.spans``), or, where they would take longer
// than the copies beside them, zeros everywhere first. Dispatch of 8192 tokens of eight choices
// takes, with those blocks, after zeros and without either: width 64 6.9, 5.6 and 2.8 us; 256
// 10.8, 12.9 and 6.8; 1024 26.1, 43.9 and 25.9; of 32768 tokens, width 64 25.4, 12.7 and 6.5; 256
// 51, 45 and 27; 1024 107, 172 and 98; 4096 tokens of two choices, width 2048, 7.4, 14.1 and 7.4.
// Every block reads all places, so beyond 2^22 of them zeros are the cheaper way again.
void zero_rest(MoveArgs& a, cudaStream_t st) {
  const int64_t pairs = int64_t(a.tokens) * a.k;
  if (pairs <= kSpan || (a.d >= 256 && pairs <= (1 << 22))) a.spans = up(pairs, kSpan);
  else RESIHP_CUDA_CHECK(cudaMemsetAsync(a.out, 0, size_t(pairs) * a.d * sizeof(__nv_bfloat16), st));
}

// As many warps as their tables (and the block's two) leave within 48 KB: 16 up to 681 experts,
// 9 at 1024.
int place_warps(int experts, int most) { return std::min(most, 49152 / ((experts + 1) * int(sizeof(int))) - 2); }
int place_bytes(int experts, int warps) { return (2 + warps) * (experts + 1) * int(sizeof(int)); }

void launch_place(const int* ids, int64_t pairs, int64_t per_block, int blocks, int start, int experts,
                  const int* counts, int* offsets, int* slots, cudaStream_t st) {
  const int warps = place_warps(experts, 16);
  RESIHP_CUDA_CHECK(launch_pdl(moe_plan_place_kernel, blocks, 32 * warps, place_bytes(experts, warps), st, ids, pairs,
                               per_block, start, experts, counts, offsets, slots));
}

// Blocks of the counting sort: at least 512 pairs each, at most one per SM (every block reads
// every block's counts).
int plan_blocks(int64_t pairs, int num_sms) { return std::max(1, std::min(num_sms, up(pairs, 512))); }

struct RouteCall {
  const void* logits;
  int64_t ld;
  int tokens, experts, k;
  bool normalize;
  int rows_per_block, blocks;
  float* weights;
  int *ids, *counts, *offsets, *slots;
};

template <typename T, int LPR, int VPT, int KMAX>
void launch_route_as(const RouteCall& c, cudaStream_t st) {
  const int warps = place_warps(c.experts, 16);
  RESIHP_CUDA_CHECK(launch_pdl(moe_route_kernel<T, LPR, VPT, KMAX>, c.blocks, 32 * warps, place_bytes(c.experts, warps), st,
                               static_cast<const T*>(c.logits), c.ld, c.tokens, c.experts, c.k, c.normalize,
                               c.rows_per_block, c.weights, c.ids, c.counts, c.offsets, c.slots));
}

// By the choices that a lane has to keep.
template <typename T, int LPR, int VPT>
void launch_route_as(const RouteCall& c, cudaStream_t st) {
  if constexpr (LPR >= 16) {
    launch_route_as<T, LPR, VPT, 16>(c, st);
  } else if constexpr (LPR == 8) {
    if (c.k <= 8) launch_route_as<T, LPR, VPT, 8>(c, st);
    else launch_route_as<T, LPR, VPT, 16>(c, st);
  } else {
    if (c.k <= 4) launch_route_as<T, LPR, VPT, 4>(c, st);
    else if (c.k <= 8) launch_route_as<T, LPR, VPT, 8>(c, st);
    else launch_route_as<T, LPR, VPT, 16>(c, st);
  }
}
static_assert(kMoeMaxChoices == 16, "the router keeps up to 16 choices");

template <typename T>
void launch_route(const RouteCall& c, cudaStream_t st) {
  if (c.experts <= 8) launch_route_as<T, 1, 8>(c, st);
  else if (c.experts <= 16) launch_route_as<T, 2, 8>(c, st);
  else if (c.experts <= 32) launch_route_as<T, 4, 8>(c, st);
  else if (c.experts <= 64) launch_route_as<T, 8, 8>(c, st);
  else if (c.experts <= 128) launch_route_as<T, 8, 16>(c, st);
  else if (c.experts <= 256) launch_route_as<T, 16, 16>(c, st);
  else if (c.experts <= 512) launch_route_as<T, 32, 16>(c, st);
  else launch_route_as<T, 32, 32>(c, st);
}

template <typename T>
void launch_route_bwd(const void* logits, int64_t ld, const float* weights, const int* ids, const float* dweights,
                      void* dlogits, int tokens, int experts, int k, bool normalize, cudaStream_t st) {
  int lpr = 1;
  while (lpr < 32 && lpr * 8 < experts) lpr <<= 1;
  auto kernel = k <= 4 ? moe_route_bwd_kernel<T, 4> : k <= 8 ? moe_route_bwd_kernel<T, 8> : moe_route_bwd_kernel<T, kMoeMaxChoices>;
  RESIHP_CUDA_CHECK(launch_pdl(kernel, up(tokens, 256 / lpr), 256, 0, st, static_cast<const T*>(logits), ld, weights,
                               ids, dweights, static_cast<T*>(dlogits), tokens, experts, k, normalize, lpr));
}

}  // namespace

int moe_blocks(int64_t pairs, int num_sms) { return plan_blocks(pairs, num_sms); }

int moe_route(const void* logits, bool bf16, int64_t ld, int tokens, int experts, int k, bool normalize,
               float* weights, int* ids, int* counts, int* offsets, int* slots, int num_sms, cudaStream_t st) {
  RESIHP_CHECK(experts >= 1 && experts <= kMoeMaxExperts, "moe_route takes 1 to ", kMoeMaxExperts, " experts");
  RESIHP_CHECK(k >= 1 && k <= kMoeMaxChoices && k <= experts, "moe_route takes 1 to ", kMoeMaxChoices,
               " choices, no more than experts");
  RESIHP_CHECK(int64_t(tokens) * k <= kMoeMaxPairs, "moe_route: tokens * k passes ", kMoeMaxPairs);
  const int64_t pairs = int64_t(tokens) * k;
  const int rows_per_block = std::max(1, up(tokens, plan_blocks(pairs, num_sms)));
  const int blocks = std::max(1, up(tokens, rows_per_block));
  const RouteCall c{logits, ld, tokens, experts, k, normalize, rows_per_block, blocks, weights, ids, counts, offsets, slots};
  if (bf16) launch_route<__nv_bfloat16>(c, st);
  else launch_route<float>(c, st);
  if (blocks == 1) return 1;
  launch_place(ids, pairs, int64_t(rows_per_block) * k, blocks, 0, experts, counts, offsets, slots, st);
  return 2;
}

void moe_route_bwd(const void* logits, bool bf16, int64_t ld, const float* weights, const int* ids,
                   const float* dweights, void* dlogits, int tokens, int experts, int k, bool normalize,
                   cudaStream_t st) {
  if (tokens == 0) return;
  if (bf16) launch_route_bwd<__nv_bfloat16>(logits, ld, weights, ids, dweights, dlogits, tokens, experts, k, normalize, st);
  else launch_route_bwd<float>(logits, ld, weights, ids, dweights, dlogits, tokens, experts, k, normalize, st);
}

void moe_plan(const int* ids, int64_t pairs, int start, int experts, int* counts, int* offsets, int* slots, int num_sms,
              cudaStream_t st) {
  RESIHP_CHECK(experts >= 1 && experts <= kMoeMaxExperts, "moe_plan takes 1 to ", kMoeMaxExperts, " experts");
  RESIHP_CHECK(pairs <= kMoeMaxPairs, "moe_plan: tokens * k passes ", kMoeMaxPairs);
  const int64_t per_block = std::max(1, up(pairs, plan_blocks(pairs, num_sms)));
  const int blocks = std::max(1, up(pairs, per_block));
  RESIHP_CUDA_CHECK(launch_pdl(moe_plan_count_kernel, blocks, 1024, (experts + 1) * int(sizeof(int)), st, ids, pairs,
                               per_block, start, experts, counts));
  launch_place(ids, pairs, per_block, blocks, start, experts, counts, offsets, slots, st);
}

void moe_scatter(const void* x, const int* slots, const int* used, void* out, int tokens, int k, int d, int* err,
                 cudaStream_t st) {
  MoveArgs a{x, nullptr, nullptr, nullptr, out, nullptr, slots, used, tokens, k, d, err, 0};
  check_move(a);
  if (tokens == 0) return;
  zero_rest(a, st);
  if (vectors(a)) launch_rows<8, 1>(moe_scatter_kernel<8, 1>, a, st);
  else launch_rows<1, 4>(moe_scatter_kernel<1, 4>, a, st);
}

void moe_gather(const void* y, const float* weights, const void* residual, const int* slots, const int* used, void* out,
                int tokens, int k, int d, int* err, int num_sms, cudaStream_t st) {
  MoveArgs a{y, nullptr, weights, residual, out, nullptr, slots, used, tokens, k, d, err, 0};
  check_move(a);
  if (tokens == 0) return;
  const bool many = tokens >= num_sms * 16;
  if (!vectors(a)) {
    launch_rows<1, 4>(moe_gather_kernel<1, 4, kTogether>, a, st);
  } else if (many && d >= 256 && k <= 32) {  // (a lane of the warp holds a choice's place)
    RESIHP_CUDA_CHECK(launch_pdl(moe_gather_warp_kernel<8, 2, 2>, up(tokens, 8), 256, 0, st, a));
  } else {
    launch_rows<8, 1>(many ? moe_gather_kernel<8, 1, 1> : moe_gather_kernel<8, 1, kTogether>, a, st);
  }
}

void moe_combine_bwd(const void* dout, const void* y, const float* weights, const int* slots, const int* used, void* dy,
                     float* dweights, int tokens, int k, int d, int* err, int num_sms, cudaStream_t st) {
  MoveArgs a{dout, y, weights, nullptr, dy, dweights, slots, used, tokens, k, d, err, 0};
  check_move(a);
  if (tokens == 0) return;
  const bool vec = vectors(a);
  const int vpr = vec ? d / 8 : d;
  const int lpr = int64_t(tokens) * k >= int64_t(num_sms) * 16 ? 32 : std::max(32, lanes_for(vpr));
  zero_rest(a, st);
  const int grid = up(int64_t(tokens) * k, 256 / lpr) + a.spans;
  auto kernel = vec ? (vpr <= lpr ? moe_combine_bwd_kernel<8, 1> : moe_combine_bwd_kernel<8, 4>) : moe_combine_bwd_kernel<1, 4>;
  RESIHP_CUDA_CHECK(launch_pdl(kernel, grid, 256, 0, st, a, lpr));
}

}  // namespace resihp
