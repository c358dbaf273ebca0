// Linear-layer products grouped by expert: one weight matrix per group, applied to a run of
// consecutive rows whose length only the device knows (tcgen05 + TMEM, as in gemm.cu).
//
//   rows    c[r, n]     = sum_k a[r, k] w[g(r)][n, k]        forward  (w read K-major)
//                                       w[g(r)][k, n]        dgrad    (w read MN-major)
//   wgrad   c[g, n, k] (+)= sum_{r in g} dy[r, n] x[r, k]    both operands read MN-major
//
// Group g owns the rows offsets[g] .. offsets[g + 1]. No group starts on a tile boundary: a
// row tile starts at its group's first row (the row coordinate of a TMA load has no
// alignment rule), reads into the next group where the group ends inside it, and stores only
// its own rows. Weights are 3-D maps, so a tile never reads into the next group's matrix:
// what lies past a matrix's edge is zero, and a next group's infinity or NaN cannot leak in.
// The weight gradient's reduction does end inside a tile: the rows of the last K block that
// belong to the next group are overwritten with zeros in shared memory before its MMAs.
// Rows behind the last group give zeros, so the output is defined everywhere.
//
// Every CTA reads the offsets itself and walks the same tile list (prefix sums of tiles per
// group in shared memory), so no second launch or host synchronisation lays it out. Offsets
// that decrease or pass the row count are clamped (and kErrBounds recorded): no value in
// them can send an access out of range.
//
// Roles as in gemm.cu: warp 0 loads, warp 1 issues the MMAs, warps 2-5 run the epilogue.
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace resihp {

namespace {

constexpr int kMaxGroups = kMoeMaxExperts;
constexpr int kBM = 128;
constexpr int kBK = 64;

struct Args {
  void* c;
  int64_t ldc;
  const int* offsets;
  int groups, rows, n, k;
  int* err;
};

template <int BN>
struct Tile {
  static constexpr int kStages = BN == 256 ? 4 : 6;
  static constexpr int kABytes = kBM * kBK * 2;
  static constexpr int kBBytes = BN * kBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kListBytes = 2 * (kMaxGroups + 2) * 4;
  static constexpr int kSmem = kStages * kStageBytes + 1024 /*align*/ + 256 /*barriers*/ + kListBytes;
  static constexpr int kTmemCols = 2 * BN;
};

// The groups' first rows and first tiles. Group ``groups`` is the rows behind the last one.
struct Lists {
  int* row;   // [groups + 2]
  int* tile;  // [groups + 2]
};

// Called by every thread of the block; TM rows per tile, ``per_row`` tiles per tile row.
__device__ __forceinline__ void build_lists(const Lists& l, const Args& g, int tm, int per_row) {
  for (int i = threadIdx.x; i <= g.groups; i += blockDim.x) l.row[i] = g.offsets[i];
  __syncthreads();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    // first rows: running maximum, clamped to 0..rows
    int carry = 0;
    bool bad = false;
    for (int e0 = 0; e0 <= g.groups; e0 += 32) {
      const int e = e0 + lane;
      const int raw = e <= g.groups ? l.row[e] : 0;
      int v = min(max(e == 0 ? 0 : raw, 0), g.rows);
      #pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v = max(v, u);
      }
      v = max(v, carry);
      if (e <= g.groups) {
        bad |= v != raw;
        l.row[e] = v;
      }
      carry = __shfl_sync(0xFFFFFFFFu, v, 31);
    }
    if (bad) record_error(g.err, kErrBounds);
    __syncwarp();
    if (lane == 0) l.row[g.groups + 1] = g.rows;
    __syncwarp();
    int sum = 0;
    for (int e0 = 0; e0 <= g.groups; e0 += 32) {
      const int e = e0 + lane;
      const int t = e <= g.groups ? (l.row[e + 1] - l.row[e] + tm - 1) / tm * per_row : 0;
      int s = t;
      #pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xFFFFFFFFu, s, o);
        if (lane >= o) s += u;
      }
      if (e <= g.groups) l.tile[e] = sum + s - t;
      sum += __shfl_sync(0xFFFFFFFFu, s, 31);
    }
    if (lane == 0) l.tile[g.groups + 1] = sum;
  }
  __syncthreads();
}

// The group of tile t (the last one that starts at or before it and is not empty).
__device__ __forceinline__ int group_of(const Lists& l, int groups, int t, int from) {
  int lo = from, hi = groups + 1;  // tile[lo] <= t < tile[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.tile[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void store_bf16(const Args& g, int row, int col0, const uint32_t (&v)[32]) {
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(g.c) + int64_t(row) * g.ldc + col0;
  #pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (col0 + 8 * j >= g.n) break;
    uint4 o;
    o.x = pack_bf16(__uint_as_float(v[8 * j]), __uint_as_float(v[8 * j + 1]));
    o.y = pack_bf16(__uint_as_float(v[8 * j + 2]), __uint_as_float(v[8 * j + 3]));
    o.z = pack_bf16(__uint_as_float(v[8 * j + 4]), __uint_as_float(v[8 * j + 5]));
    o.w = pack_bf16(__uint_as_float(v[8 * j + 6]), __uint_as_float(v[8 * j + 7]));
    *reinterpret_cast<uint4*>(out + 8 * j) = o;
  }
}

// ---- rows: forward and input gradient --------------------------------------------------

template <int BN, bool W_MN>
__global__ void __launch_bounds__(192, 1)
    grouped_rows_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_w, Args g) {
  pdl_enter();
  using S = Tile<BN>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024 - (raw & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * S::kStageBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  Lists l;
  l.row = reinterpret_cast<int*>(smem + kStages * S::kStageBytes + 256);
  l.tile = l.row + kMaxGroups + 2;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int tiles_n = (g.n + BN - 1) / BN;
  const int kblocks = (g.k + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 4);
    }
    fence_barrier_init();
    tma_prefetch(&tma_a);
    tma_prefetch(&tma_w);
  }
  if (warp == 1) tmem_alloc(tmem_slot, S::kTmemCols);
  build_lists(l, g, kBM, tiles_n);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int work = l.tile[g.groups];        // tiles with a product
  const int tiles = l.tile[g.groups + 1];   // and those of the rows behind the last group

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, e = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < work && ok; t += gridDim.x) {
        e = group_of(l, g.groups, t, e);
        int tm, tn;
        tile_coords(t - l.tile[e], (l.tile[e + 1] - l.tile[e]) / tiles_n, tiles_n, tm, tn);
        const int m0 = l.row[e] + tm * kBM, n0 = tn * BN;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1, g.err, kErrTmaWait)) { ok = false; break; }
          uint8_t* sa = smem + s * S::kStageBytes;
          uint8_t* sb = sa + S::kABytes;
          mbar_expect_tx(&full[s], S::kStageBytes);
          const int k0 = kb * kBK;
          tma_load_2d(sa, &tma_a, &full[s], k0, m0, g.err);
          if (W_MN) {
            #pragma unroll
            for (int c = 0; c < BN / 64; ++c) tma_load_3d(sb + c * 8192, &tma_w, &full[s], n0 + 64 * c, k0, e, g.err);
          } else {
            tma_load_3d(sb, &tma_w, &full[s], k0, n0, e, g.err);
          }
          if (++s == kStages) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_bf16_f32(kBM, BN, 0, W_MN ? 1 : 0);
      int s = 0, i = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < work && ok; t += gridDim.x, ++i) {
        const int a = i & 1;
        if (!mbar_wait(&acc_empty[a], ((i >> 1) & 1) ^ 1, g.err, kErrMmaWait)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + a * BN;
        if (!tmem_span_ok(d, tmem_base, S::kTmemCols, BN, g.err)) break;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&full[s], ph, g.err, kErrMmaWait)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * S::kStageBytes);
          const uint32_t sb = sa + S::kABytes;
          #pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk) {
            const uint64_t da = smem_desc_sw128(sa + kk * 32, 16, 1024);
            const uint64_t db = W_MN ? smem_desc_sw128(sb + kk * 2048, 8192, 1024)
                                     : smem_desc_sw128(sb + kk * 32, 16, 1024);
            umma_bf16(d, da, db, idesc, (kb | kk) != 0);
          }
          umma_commit(&empty[s]);
          if (++s == kStages) { s = 0; ph ^= 1; }
        }
        umma_commit(&acc_full[a]);
      }
    }
  } else {
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    int i = 0, e = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
      e = group_of(l, g.groups, t, e);
      int tm, tn;
      tile_coords(t - l.tile[e], (l.tile[e + 1] - l.tile[e]) / tiles_n, tiles_n, tm, tn);
      const int row = l.row[e] + tm * kBM + q * 32 + lane;
      const bool row_ok = row < l.row[e + 1];
      if (e == g.groups) {  // behind the last group: zeros
        const uint32_t zero[32] = {};
        for (int c = 0; c < BN / 32; ++c)
          if (row_ok && tn * BN + c * 32 < g.n) store_bf16(g, row, tn * BN + c * 32, zero);
        continue;
      }
      const int a = i & 1;
      if (!mbar_wait(&acc_full[a], (i >> 1) & 1, g.err, kErrEpiWait)) break;
      tc_fence_after();
      #pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t v[32];
        const uint32_t ta = tmem_base + a * BN + c * 32 + (uint32_t(q * 32) << 16);
        if (!tmem_span_ok(ta, tmem_base, S::kTmemCols, 32, g.err)) continue;
        tmem_ld32(ta, v);
        tmem_wait_ld();
        const int col0 = tn * BN + c * 32;
        if (row_ok && col0 < g.n) store_bf16(g, row, col0, v);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[a]);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// ---- weight gradient --------------------------------------------------------------------

// Tile rows are the group's output features (n), tile columns its input features (k).
template <int BN, bool ACC>
__global__ void __launch_bounds__(192, 1)
    grouped_wgrad_kernel(const __grid_constant__ CUtensorMap tma_dy, const __grid_constant__ CUtensorMap tma_x, Args g) {
  pdl_enter();
  using S = Tile<BN>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024 - (raw & 1023)) & 1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * S::kStageBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  Lists l;
  l.row = reinterpret_cast<int*>(smem + kStages * S::kStageBytes + 256);
  l.tile = l.row + kMaxGroups + 2;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int tiles_m = (g.n + kBM - 1) / kBM, tiles_n = (g.k + BN - 1) / BN;
  const int per_group = tiles_m * tiles_n;
  const int tiles = g.groups * per_group;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 4);
    }
    fence_barrier_init();
    tma_prefetch(&tma_dy);
    tma_prefetch(&tma_x);
  }
  if (warp == 1) tmem_alloc(tmem_slot, S::kTmemCols);
  build_lists(l, g, kBK, 1);  // "tiles": the group's K blocks
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int e = t / per_group;
        int tm, tn;
        tile_coords(t - e * per_group, tiles_m, tiles_n, tm, tn);
        const int kblocks = l.tile[e + 1] - l.tile[e];
        const int m0 = tm * kBM, n0 = tn * BN;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&empty[s], ph ^ 1, g.err, kErrTmaWait)) { ok = false; break; }
          uint8_t* sa = smem + s * S::kStageBytes;
          uint8_t* sb = sa + S::kABytes;
          mbar_expect_tx(&full[s], S::kStageBytes);
          const int r0 = l.row[e] + kb * kBK;
          #pragma unroll
          for (int c = 0; c < kBM / 64; ++c) tma_load_2d(sa + c * 8192, &tma_dy, &full[s], m0 + 64 * c, r0, g.err);
          #pragma unroll
          for (int c = 0; c < BN / 64; ++c) tma_load_2d(sb + c * 8192, &tma_x, &full[s], n0 + 64 * c, r0, g.err);
          if (++s == kStages) { s = 0; ph ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // the whole warp walks the stages (it zeroes a cut K block together); lane 0 issues
    constexpr uint32_t idesc = idesc_bf16_f32(kBM, BN, 1, 1);
    int s = 0, i = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const int e = t / per_group;
      const int kblocks = l.tile[e + 1] - l.tile[e];
      if (kblocks == 0) continue;
      const int size = l.row[e + 1] - l.row[e];
      const int a = i & 1;
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(&acc_empty[a], ((i >> 1) & 1) ^ 1, g.err, kErrMmaWait))) break;
      ++i;
      tc_fence_after();
      const uint32_t d = tmem_base + a * BN;
      if (!tmem_span_ok(d, tmem_base, S::kTmemCols, BN, g.err)) break;
      for (int kb = 0; kb < kblocks; ++kb) {
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(&full[s], ph, g.err, kErrMmaWait))) { ok = false; break; }
        const int valid = min(kBK, size - kb * kBK);
        const int steps = (valid + 15) / 16;
        uint8_t* sa_p = smem + s * S::kStageBytes;
        if (valid < 16 * steps) {
          // MN-major chunks are 64 rows of 128 bytes: rows valid .. 16 * steps hold the
          // next group's rows (both operands: 0 * inf would not be 0)
          const int bytes = (16 * steps - valid) * 128;
          #pragma unroll 1
          for (int c = 0; c < (kBM + BN) / 64; ++c)
            for (int b = lane * 16; b < bytes; b += 512)
              *reinterpret_cast<uint4*>(sa_p + c * 8192 + valid * 128 + b) = make_uint4(0, 0, 0, 0);
          fence_proxy_async();
          __syncwarp();
        }
        if (lane == 0) {
          tc_fence_after();
          const uint32_t sa = smem_u32(sa_p);
          const uint32_t sb = sa + S::kABytes;
          for (int kk = 0; kk < steps; ++kk)
            umma_bf16(d, smem_desc_sw128(sa + kk * 2048, 8192, 1024), smem_desc_sw128(sb + kk * 2048, 8192, 1024),
                      idesc, (kb | kk) != 0);
          umma_commit(&empty[s]);
        }
        __syncwarp();
        if (++s == kStages) { s = 0; ph ^= 1; }
      }
      if (lane == 0) umma_commit(&acc_full[a]);
      __syncwarp();
    }
  } else {
    const int q = warp & 3;
    int i = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      const int e = t / per_group;
      const bool empty_group = l.tile[e + 1] == l.tile[e];
      if (empty_group && ACC) continue;
      int tm, tn;
      tile_coords(t - e * per_group, tiles_m, tiles_n, tm, tn);
      const int row = tm * kBM + q * 32 + lane;
      const bool row_ok = row < g.n;
      float* out = static_cast<float*>(g.c) + (int64_t(e) * g.n + row) * g.k;
      const int a = i & 1;
      if (!empty_group) {
        if (!mbar_wait(&acc_full[a], (i >> 1) & 1, g.err, kErrEpiWait)) break;
        ++i;
        tc_fence_after();
      }
      #pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t v[32];
        if (empty_group) {
          #pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0u;
        } else {
          const uint32_t ta = tmem_base + a * BN + c * 32 + (uint32_t(q * 32) << 16);
          if (!tmem_span_ok(ta, tmem_base, S::kTmemCols, 32, g.err)) continue;
          tmem_ld32(ta, v);
          tmem_wait_ld();
        }
        const int col0 = tn * BN + c * 32;
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (!row_ok || col0 + 4 * j >= g.k) break;
          const float4 o = make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]),
                                       __uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3]));
          if (ACC) red_add_v4(out + col0 + 4 * j, o);
          else *reinterpret_cast<float4*>(out + col0 + 4 * j) = o;
        }
      }
      if (!empty_group) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[a]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// ---- launches ---------------------------------------------------------------------------

int num_sms() {
  static int counts[64] = {0};
  int dev = 0;
  RESIHP_CUDA_CHECK(cudaGetDevice(&dev));
  if (counts[dev] == 0) RESIHP_CUDA_CHECK(cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev));
  return counts[dev];
}

template <typename Kernel>
void launch(Kernel kernel, int smem, int64_t tiles, const CUtensorMap& ta, const CUtensorMap& tb, const Args& g,
            cudaStream_t st) {
  RESIHP_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int grid = int(std::min<int64_t>(tiles, num_sms()));
  RESIHP_CUDA_CHECK(launch_pdl(kernel, grid, 192, smem, st, ta, tb, g));
}

void check_shape(const GroupedShape& s) {
  RESIHP_CHECK(s.groups >= 1 && s.groups <= kMaxGroups, "grouped products take 1 to ", kMaxGroups, " groups");
  RESIHP_CHECK(s.n >= 8 && s.k >= 8 && s.n % 8 == 0 && s.k % 8 == 0,
               "grouped products need widths that are multiples of 8 (16-byte vectors)");
  RESIHP_CHECK(s.rows >= 0, "grouped products: negative row count");
}

}  // namespace

void grouped_rows(const void* a, int64_t lda, const void* w, int64_t ldw, int64_t w_group, bool w_mn, void* c,
                  int64_t ldc, const GroupedShape& s, int* err, cudaStream_t st) {
  check_shape(s);
  if (s.rows == 0) return;
  RESIHP_CHECK(reinterpret_cast<uintptr_t>(c) % 16 == 0 && ldc % 8 == 0, "grouped output must be 16-byte aligned");
  constexpr int BN = 128;
  const int64_t tiles_n = (s.n + BN - 1) / BN;
  const int64_t most = (int64_t(s.rows) + kBM - 1) / kBM + s.groups + 1;  // tile rows, if every group cuts one
  RESIHP_CHECK(most * tiles_n <= INT32_MAX, "grouped products: too many tiles");
  const CUtensorMap ta = make_tma_2d_bf16(a, s.rows, s.k, lda, 64, kBM);
  const CUtensorMap tw = w_mn ? make_tma_3d_bf16(w, s.groups, s.k, s.n, ldw, w_group, 64, 64)
                              : make_tma_3d_bf16(w, s.groups, s.n, s.k, ldw, w_group, 64, BN);
  const Args g{c, ldc, s.offsets, s.groups, s.rows, s.n, s.k, err};
  using S = Tile<BN>;
  if (w_mn) launch(grouped_rows_kernel<BN, true>, S::kSmem, most * tiles_n, ta, tw, g, st);
  else launch(grouped_rows_kernel<BN, false>, S::kSmem, most * tiles_n, ta, tw, g, st);
}

void grouped_wgrad(const void* dy, int64_t lddy, const void* x, int64_t ldx, float* c, bool accumulate,
                   const GroupedShape& s, int* err, cudaStream_t st) {
  check_shape(s);
  RESIHP_CHECK(reinterpret_cast<uintptr_t>(c) % 16 == 0, "grouped weight gradient must be 16-byte aligned");
  if (s.rows == 0) {
    if (!accumulate) RESIHP_CUDA_CHECK(cudaMemsetAsync(c, 0, sizeof(float) * size_t(s.groups) * s.n * s.k, st));
    return;
  }
  constexpr int BN = 128;
  const int64_t tiles = int64_t(s.groups) * ((s.n + kBM - 1) / kBM) * ((s.k + BN - 1) / BN);
  RESIHP_CHECK(tiles <= INT32_MAX, "grouped products: too many tiles");
  const CUtensorMap ta = make_tma_2d_bf16(dy, s.rows, s.n, lddy, 64, 64);
  const CUtensorMap tb = make_tma_2d_bf16(x, s.rows, s.k, ldx, 64, 64);
  const Args g{c, 0, s.offsets, s.groups, s.rows, s.n, s.k, err};
  using S = Tile<BN>;
  if (accumulate) launch(grouped_wgrad_kernel<BN, true>, S::kSmem, tiles, ta, tb, g, st);
  else launch(grouped_wgrad_kernel<BN, false>, S::kSmem, tiles, ta, tb, g, st);
}

}  // namespace resihp
