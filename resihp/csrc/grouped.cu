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
// The weight gradient's reduction does end inside a tile: the rows of its last MMA step that
// belong to the next group are overwritten with zeros in shared memory first.
// Rows behind the last group give zeros, so the output is defined everywhere.
//
// Every CTA reads the offsets itself and walks the same tile list (prefix sums of tiles per
// group in shared memory), so no second launch or host synchronisation lays it out. Offsets
// that decrease or pass the row count are clamped (and kErrBounds recorded): no value in
// them can send an access out of range.
//
// Roles as in gemm.cu, on CTA pairs: warp 0 loads, the leader's warp 1 issues the MMAs, the
// others run the epilogue. The loading and issuing warps walk their loops whole and one lane of
// them issues: their counters, addresses and descriptors are then the same in all lanes, which
// the instructions want, and a block of 256 x 256 x 64 is issued in less than the 512 cycles
// its MMAs take (from inside a branch on the lane it took 1000: 1234 TF/s forward, then 1366).
#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace resihp {

namespace {

constexpr int kMaxGroups = kMoeMaxExperts;

struct Args {
  void* c;
  int64_t ldc;
  const int* offsets;
  int groups, rows, n, k;
  unsigned* pace;  // rows: see pace_pairs; nullptr: pairs run freely
  int* err;
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

// ---- rows: forward and input gradient --------------------------------------------------
//
// The product is computed transposed, c^T = w a^T: the weights' output features are the MMA's
// M (256 per CTA pair, 128 per CTA), the group's rows its N. N is an operand of each MMA, a
// multiple of 32 up to TN, so a group whose length is no multiple of a tile costs what its
// rows cost (at 8 groups of about 1024 rows, 256-row M tiles would do 12 % more work), and a
// handful of rows costs one narrow MMA per K step while the weights stream past. A group of
// more than TN rows is cut into equal parts, not into full tiles and a rest.
//
// Many rows: bound by the tensor cores, and in long products by the power cap: 8192 rows of
// eight groups, 2048 > 11008, take 268 us forward and 280 backward (1376 and 1319 TF/s of the
// 1643 a library product reaches in a burst, 1397 sustained). Few rows: bound by reading the
// weights: 16 rows, same weights, 60 us (6.0 TB/s of the 6.5 a copy reaches).
//
// One accumulator takes the whole depth, with the truncating additions that the weight gradient
// below cuts short: at most 2e-5 of the norm at these depths, where the output's rounding to bf16 is
// 1.7e-3. It moves 0.1 % of the outputs (k 2048) to 0.8 % (k 13824) across a rounding's border.

constexpr int kBK = 64;

template <int TN>
struct RowTile {
  static constexpr int kWBytes = 128 * kBK * 2;         // this CTA's 128 features
  static constexpr int kABytes = TN / 2 * kBK * 2;      // this CTA's half of the rows
  static constexpr int kStageBytes = kWBytes + kABytes;
  static constexpr int kStages = TN == 256 ? 6 : 8;
  static constexpr int kListBytes = 2 * (kMaxGroups + 2) * 4;
  static constexpr int kSmem = kStages * kStageBytes + 1024 /*align*/ + 256 /*barriers*/ + kListBytes;
  static constexpr int kTmemCols = 2 * TN;
  static_assert(kSmem <= 232448, "grouped stages exceed the shared memory of a CTA");
  static_assert((2 * kStages + 4) * 8 + 4 <= 256, "grouped barriers exceed their area");
};

// Rows of a tile as the pair MMA takes them: its N goes in steps of 32.
__device__ __forceinline__ int mma_rows(int rows) { return (rows + 31) & ~31; }

struct RowSpan {
  int row0, rows, f0;  // first row, row count and first output feature of a tile
};

template <int TN>
__device__ __forceinline__ RowSpan span_of(const Lists& l, int e, int t, int tiles_f) {
  const int size = l.row[e + 1] - l.row[e];
  const int parts = (l.tile[e + 1] - l.tile[e]) / tiles_f;
  int tm, tf;
  tile_coords(t - l.tile[e], parts, tiles_f, tm, tf);
  const int each = mma_rows((size + parts - 1) / parts);  // parts * each >= size, each <= TN
  return RowSpan{l.row[e] + tm * each, min(each, size - tm * each), tf * 256};
}

// Pacing. The tiles under way at one time share operand tiles: 74 pairs read about 17 panels of
// 256 rows or features at once. Pairs that drift apart by more than L2 holds of those read the
// same bytes again from memory: 16384 rows, 13824 > 5120, eight uneven groups, brought 7.7 GB
// in where 1.6 are needed, and the last pair ended 18 % after the first. Where the panels of a
// round pass half of L2 (k from 7168 on) every pair therefore counts itself in each 64 K
// blocks, and waits a moment while the pairs' steps add up to fewer than its own times the number
// of pairs. That bounds how far a pair runs ahead of the average, not of the slowest: one straggler
// holds nobody up. 1122 -> 1220 TF/s there under the power cap; at k = 5504 and 11008
// (8192 rows), the only other depths it was timed at, it neither gains nor costs.
constexpr int kPaceBlocks = 64;
constexpr int kPaceDepth = 7168;
constexpr uint64_t kPaceNs = 20000;

// One lane of every pair, at each step. False once the others take too long (pairs that are not
// resident, a device that is shared): the pair then runs freely, as nothing but time depends on
// it.
__device__ __forceinline__ bool pace_pairs(unsigned* count, unsigned step, unsigned pairs) {
  atomicAdd(count, 1u);
  if (step == 0) return true;
  const uint64_t start = globaltimer();
  while (*reinterpret_cast<volatile unsigned*>(count) < step * pairs) {
    if (globaltimer() - start > kPaceNs) return false;
    __nanosleep(64);
  }
  return true;
}

template <int TN, bool W_MN>
__global__ void __launch_bounds__(192, 1)
    grouped_rows_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_a, Args g) {
  pdl_enter();
  using S = RowTile<TN>;
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

  const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0);  // uniform for the compiler too
  const int lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();  // 0: leader, 1: peer
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles_f = (g.n + 255) / 256;
  const int kblocks = (g.k + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 8);
    }
    fence_barrier_init();
    tma_prefetch(&tma_w);
    tma_prefetch(&tma_a);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, S::kTmemCols);
  build_lists(l, g, TN, tiles_f);
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers initialised and TMEM allocated before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int work = l.tile[g.groups];        // tiles with a product
  const int tiles = l.tile[g.groups + 1];   // and those of the rows behind the last group

  if (warp == 0) {
    // the whole warp walks, one lane issues
    const uint32_t issue = elect_one(), lead = cta == 0 ? issue : 0u;
    const uint32_t sbase = smem_u32(smem), fbase = smem_u32(full), fleader = mapa_shared(full, 0);
    int s = 0, e = 0;
    uint32_t ph = 0;
    bool ok = true;
    bool paced = g.pace != nullptr;  // the same in all lanes
    unsigned step = 0;
    for (int t = pair; t < work && ok; t += pairs) {
      paced = paced && t - pair + pairs <= work;  // not in the last round, which some pairs sit out
      e = group_of(l, g.groups, t, e);
      const RowSpan p = span_of<TN>(l, e, t, tiles_f);
      // each CTA brings its features and its half of the MMA's N rows
      const int f0 = p.f0 + int(cta) * 128;
      const int r0 = __shfl_sync(0xFFFFFFFFu, p.row0 + int(cta) * (mma_rows(p.rows) >> 1), 0);
      const int plane = __shfl_sync(0xFFFFFFFFu, e, 0);
      for (int kb = 0; kb < kblocks; ++kb) {
        if (paced && kb % kPaceBlocks == 0) {
          bool in_time = true;
          if (lead) in_time = pace_pairs(g.pace, step, unsigned(pairs));
          paced = __all_sync(0xFFFFFFFFu, in_time);
          ++step;
        }
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(&empty[s], ph ^ 1, g.err, kErrTmaWait))) { ok = false; break; }
        const uint32_t sw = sbase + s * S::kStageBytes, bar = fleader + s * 8;
        mbar_expect_tx_if(lead, fbase + s * 8, 2 * S::kStageBytes);  // both CTAs' parts
        const int k0 = kb * kBK;
        if (W_MN) {
          tma_load_3d_pair_if(issue, sw, &tma_w, bar, f0, k0, plane, g.err);
          tma_load_3d_pair_if(issue, sw + 8192, &tma_w, bar, f0 + 64, k0, plane, g.err);
        } else {
          tma_load_3d_pair_if(issue, sw, &tma_w, bar, k0, f0, plane, g.err);
        }
        tma_load_2d_pair_if(issue, sw + S::kWBytes, &tma_a, bar, k0, r0, g.err);
        if (++s == kStages) { s = 0; ph ^= 1; }
      }
    }
    // Producer tail: wait until the leader has released every stage, so no pair-MMA commit can
    // arrive on this CTA's barriers after it exits.
    for (int j = 0; j < kStages && ok; ++j) {
      if (!mbar_wait(&empty[s], ph ^ 1, g.err, kErrTmaWait)) break;
      if (++s == kStages) { s = 0; ph ^= 1; }
    }
  } else if (warp == 1) {
    if (cta == 0) {  // the whole warp walks, one lane issues
      const uint32_t issue = elect_one();
      const uint32_t sbase = smem_u32(smem), bar0 = smem_u32(empty), bar1 = mapa_shared(empty, 1);
      const uint32_t done0 = smem_u32(acc_full), done1 = mapa_shared(acc_full, 1);
      int s = 0, i = 0, e = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int t = pair; t < work && ok; t += pairs, ++i) {
        e = group_of(l, g.groups, t, e);
        const int n = __shfl_sync(0xFFFFFFFFu, mma_rows(span_of<TN>(l, e, t, tiles_f).rows), 0);
        const uint32_t idesc = idesc_bf16_f32(256, n, W_MN ? 1 : 0, 0);
        const int a = i & 1;
        if (!__all_sync(0xFFFFFFFFu, mbar_wait_cluster(&acc_empty[a], ((i >> 1) & 1) ^ 1, g.err, kErrMmaWait))) break;
        const uint32_t d = tmem_base + a * TN;
        if (!tmem_span_ok(d, tmem_base, S::kTmemCols, n, g.err)) break;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!__all_sync(0xFFFFFFFFu, mbar_wait(&full[s], ph, g.err, kErrMmaWait))) { ok = false; break; }
          tc_fence_after();
          // the descriptors' address field counts 16-byte units: a K step adds to it
          const uint32_t sw = sbase + s * S::kStageBytes;
          const uint64_t dw = W_MN ? smem_desc_sw128(sw, 8192, 1024) : smem_desc_sw128(sw, 16, 1024);
          const uint64_t da = smem_desc_sw128(sw + S::kWBytes, 16, 1024);
          #pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk)
            umma_bf16_pair_if(issue, d, dw + kk * (W_MN ? 2048 / 16 : 32 / 16), da + kk * (32 / 16), idesc,
                              (kb | kk) != 0);
          umma_commit_pair_if(issue, bar0 + s * 8);
          umma_commit_pair_if(issue, bar1 + s * 8);
          if (++s == kStages) { s = 0; ph ^= 1; }
        }
        if (!ok) break;
        umma_commit_pair_if(issue, done0 + a * 8);
        umma_commit_pair_if(issue, done1 + a * 8);
      }
    }
  } else {
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    const uint32_t acc_empty_leader0 = mapa_shared(&acc_empty[0], 0);
    const uint32_t acc_empty_leader1 = mapa_shared(&acc_empty[1], 0);
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(g.c);
    int i = 0, e = 0;
    for (int t = pair; t < tiles; t += pairs, ++i) {
      e = group_of(l, g.groups, t, e);
      const RowSpan p = span_of<TN>(l, e, t, tiles_f);
      const int fc = p.f0 + int(cta) * 128;  // this CTA's first feature
      if (e == g.groups) {  // behind the last group: zeros, 128 features of a row per half warp
        const int f = fc + (lane & 15) * 8;
        for (int r = q * 2 + (lane >> 4); r < p.rows; r += 8)
          if (f < g.n) *reinterpret_cast<uint4*>(out + int64_t(p.row0 + r) * g.ldc + f) = make_uint4(0, 0, 0, 0);
        continue;
      }
      const int a = i & 1;
      if (!mbar_wait(&acc_full[a], (i >> 1) & 1, g.err, kErrEpiWait)) break;
      tc_fence_after();
      // Lane f holds feature f of 32 rows. Neighbouring lanes swap one value per two rows, so
      // that each stores two features of one row: a warp's store covers 64 bytes of two rows.
      const int f = fc + q * 32 + (lane & ~1);
      const bool odd = lane & 1;
      __nv_bfloat16* base = out + int64_t(p.row0 + (odd ? 1 : 0)) * g.ldc + f;
      #pragma unroll 1
      for (int c = 0; c < p.rows; c += 32) {
        uint32_t v[32];
        const uint32_t ta = tmem_base + a * TN + c + (uint32_t(q * 32) << 16);
        if (!tmem_span_ok(ta, tmem_base, S::kTmemCols, 32, g.err)) continue;
        tmem_ld32(ta, v);
        tmem_wait_ld();
        #pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, odd ? v[j] : v[j + 1], 1);
          const uint32_t o = odd ? pack_bf16(__uint_as_float(got), __uint_as_float(v[j + 1]))
                                 : pack_bf16(__uint_as_float(v[j]), __uint_as_float(got));
          if (c + j + (odd ? 1 : 0) < p.rows && f < g.n)
            *reinterpret_cast<uint32_t*>(base + int64_t(c + j) * g.ldc) = o;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(a == 0 ? acc_empty_leader0 : acc_empty_leader1);
    }
  }

  tc_fence_before();
  cluster_sync();  // no CTA leaves while its pair may still touch its barriers or TMEM
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, S::kTmemCols);
  }
}

// ---- weight gradient --------------------------------------------------------------------
//
// Tile: 256 output features (n) x 256 input features (k) of one group on a CTA pair, reduced
// over the group's rows in blocks of 64. The tensor cores add into an accumulator with
// truncation, so a long sum drifts: off by 1e-6 of its norm after 1024 rows, 4e-6 after 4096,
// 1.9e-5 after 16384 (an fp32 library product: 3e-7 to 6e-7). Every 512 rows the accumulator is
// therefore handed to the epilogue, which adds it to fp32 registers with rounding, while the
// MMAs go on in the other accumulator: 4.8e-7 at every length, for 3 % of the rate (1222
// against 1255 TF/s, two groups of 8192 rows; every 256 rows 2.7e-7 at 1125). Eight epilogue
// warps per CTA keep 128 columns of a row per thread. The finished tile leaves through shared
// memory as bulk stores or bulk additions (whole 128-byte runs, clipped at the matrix's edges
// by the map): each element is added to once per launch, so no order can change the sum.
// 8192 rows of eight groups, 2048 x 11008: 322 us written, 374 added to what is there (721 MB
// of fp32, of which the sums alone would take 110 us and 220; the MMAs 270). As a bf16 gradient,
// rounded once from the fp32 sum, 283 us; written in fp32 and cast by another kernel 440. With the
// GPU at its power cap, after other long products, 360, 410 to 430 and 265 to 300.
//
// A group's last block holds rows of the next group where its length is no multiple of 64.
// Steps of 16 rows past the end are not issued; rows past the end inside the last step are
// zeroed in shared memory by warp 2 of each CTA. Such a block's loads complete on the CTA's own
// ``cut`` barrier, and the leader's MMAs wait for both CTAs' arrivals on ``zeroed``.

constexpr int kWChunk = 8;       // blocks per accumulator
constexpr int kWStages = 5;
constexpr int kWThreads = 384;   // dy producer, MMA, zeroing, eight epilogue warps, x producer
struct WgradTile {
  static constexpr int kChunkBytes = 64 * kBK * 2;  // 64 columns of a block, MN-major
  static constexpr int kABytes = 2 * kChunkBytes;   // this CTA's 128 columns of dy, then of x
  static constexpr int kStageBytes = 4 * kChunkBytes;
  static constexpr int kOutBytes = 32 * 32 * 4;  // per epilogue warp: 32 x 32 fp32
  static constexpr int kListBytes = 2 * (kMaxGroups + 2) * 4;
  static constexpr int kSmem = kWStages * kStageBytes + 8 * kOutBytes + 1024 + 256 + kListBytes;
  static constexpr int kTmemCols = 512;
  static_assert(kSmem <= 232448, "grouped wgrad stages exceed the shared memory of a CTA");
  static_assert((4 * kWStages + 4) * 8 + 4 <= 256, "grouped wgrad barriers exceed their area");
};

// Tile t of a group of ``blocks`` blocks. Groups of one accumulator spend their time writing, and
// go along the gradient's rows, so that what is written together lies together; longer ones go
// eight tile rows at a time, so that tiles running together share operands. Four runs of each,
// in turn: 16 rows, 2048 x 11008, written 127 to 134 us against 129 to 175, accumulated 251 to
// 258 against 252 to 282; 64 groups of 94 rows, 1024 x 1416, written 92.7 against 93 to 99,
// accumulated 130 against 131 to 137. Two groups of 8192 rows, 13824 x 5120, accumulated 2250 us
// along the rows and 2120 in groups of eight.
__device__ __forceinline__ void wgrad_coords(int t, int blocks, int tiles_m, int tiles_n, int& tm, int& tn) {
  if (blocks <= kWChunk) {
    tm = t / tiles_n;
    tn = t - tm * tiles_n;
  } else {
    tile_coords(t, tiles_m, tiles_n, tm, tn);
  }
}

// Rows of a group's block kb that belong to it, and whether its last MMA step is cut.
__device__ __forceinline__ int valid_rows(int size, int kb) { return min(kBK, size - kb * kBK); }
__device__ __forceinline__ bool is_cut(int valid) { return (valid & 15) != 0; }

template <bool ACC, bool BF16>
__global__ void __launch_bounds__(kWThreads, 1)
    grouped_wgrad_kernel(const __grid_constant__ CUtensorMap tma_dy, const __grid_constant__ CUtensorMap tma_x,
                         const __grid_constant__ CUtensorMap tma_c, Args g) {
  pdl_enter();
  using S = WgradTile;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024 - (raw & 1023)) & 1023);
  uint8_t* staging = smem + kWStages * S::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + 8 * S::kOutBytes);
  uint64_t* empty = full + kWStages;
  uint64_t* cut = empty + kWStages;
  uint64_t* zeroed = cut + kWStages;
  uint64_t* acc_full = zeroed + kWStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  Lists l;
  l.row = reinterpret_cast<int*>(staging + 8 * S::kOutBytes + 256);
  l.tile = l.row + kMaxGroups + 2;

  const int warp = __shfl_sync(0xFFFFFFFFu, int(threadIdx.x) >> 5, 0);  // uniform for the compiler too
  const int lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank();  // 0: leader, 1: peer
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles_m = (g.n + 255) / 256, tiles_n = (g.k + 255) / 256;
  const int per_group = tiles_m * tiles_n;
  const int tiles = g.groups * per_group;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kWStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&cut[s], 1);
      mbar_init(&zeroed[s], 2);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 16);
    }
    fence_barrier_init();
    tma_prefetch(&tma_dy);
    tma_prefetch(&tma_x);
    tma_prefetch(&tma_c);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, S::kTmemCols);
  build_lists(l, g, kBK, 1);  // "tiles": the group's row blocks
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers initialised and TMEM allocated before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0 || warp == 11) {
    // Two producers, one per operand: a load costs its warp about 120 cycles, and four of them
    // per block would pace the MMAs (512 cycles; 8192 rows, 2048 x 11008, eight groups, written:
    // 370 us with one producer, 345 with two, then). The whole warp walks, one lane issues.
    const bool second = warp == 11;
    const uint32_t issue = elect_one(), lead = cta == 0 && !second ? issue : 0u, own = second ? 0u : issue;
    const CUtensorMap* map = second ? &tma_x : &tma_dy;
    const int part = second ? S::kABytes : 0;
    const uint32_t sbase = smem_u32(smem), fbase = smem_u32(full), fleader = mapa_shared(full, 0);
    const uint32_t cbase = smem_u32(cut), cown = mapa_shared(cut, cta);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int e = t / per_group;
      int tm, tn;
      wgrad_coords(t - e * per_group, l.tile[e + 1] - l.tile[e], tiles_m, tiles_n, tm, tn);
      int r0 = __shfl_sync(0xFFFFFFFFu, l.row[e], 0);
      int left = __shfl_sync(0xFFFFFFFFu, l.row[e + 1], 0) - r0;
      const int c0 = (second ? tn : tm) * 256 + int(cta) * 128;
      for (; left > 0; left -= kBK, r0 += kBK) {
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(&empty[s], ph ^ 1, g.err, kErrTmaWait))) { ok = false; break; }
        uint32_t bar = fleader + s * 8;
        if (left < kBK && is_cut(left)) {
          mbar_arrive_if(lead, fbase + s * 8);
          mbar_expect_tx_if(own, cbase + s * 8, S::kStageBytes);
          bar = cown + s * 8;
        } else {
          mbar_expect_tx_if(lead, fbase + s * 8, 2 * S::kStageBytes);  // both CTAs' halves
        }
        const uint32_t dst = sbase + s * S::kStageBytes + part;
        tma_load_2d_pair_if(issue, dst, map, bar, c0, r0, g.err);
        tma_load_2d_pair_if(issue, dst + S::kChunkBytes, map, bar, c0 + 64, r0, g.err);
        if (++s == kWStages) { s = 0; ph ^= 1; }
      }
    }
    // Producer tail: every stage released, so no commit can arrive after this CTA exits.
    for (int j = 0; j < kWStages && ok; ++j) {
      if (!mbar_wait(&empty[s], ph ^ 1, g.err, kErrTmaWait)) break;
      if (++s == kWStages) { s = 0; ph ^= 1; }
    }
  } else if (warp == 1) {
    if (cta == 0) {  // the whole warp walks, one lane issues
      const uint32_t issue = elect_one();
      constexpr uint32_t idesc = idesc_bf16_f32(256, 256, 1, 1);
      const uint32_t sbase = smem_u32(smem), bar0 = smem_u32(empty), bar1 = mapa_shared(empty, 1);
      const uint32_t done0 = smem_u32(acc_full), done1 = mapa_shared(acc_full, 1);
      int s = 0, i = 0;
      uint32_t ph = 0, zph = 0;  // zph: a parity bit per stage
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        const int e = t / per_group;
        int left = __shfl_sync(0xFFFFFFFFu, l.row[e + 1] - l.row[e], 0);  // rows still to add
        while (left > 0 && ok) {  // one accumulator
          const int a = i & 1;
          const uint32_t d = tmem_base + a * 256;
          if (!__all_sync(0xFFFFFFFFu, mbar_wait_cluster(&acc_empty[a], ((i >> 1) & 1) ^ 1, g.err, kErrMmaWait)) ||
              !tmem_span_ok(d, tmem_base, S::kTmemCols, 256, g.err)) {
            ok = false;
            break;
          }
          uint32_t onto = 0;
          for (int kb = 0; kb < kWChunk && left > 0; ++kb) {
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(&full[s], ph, g.err, kErrMmaWait))) { ok = false; break; }
            const uint32_t sa = sbase + s * S::kStageBytes;
            const uint64_t da = smem_desc_sw128(sa, S::kChunkBytes, 1024);
            const uint64_t db = smem_desc_sw128(sa + S::kABytes, S::kChunkBytes, 1024);
            if (left >= kBK) {
              tc_fence_after();
              #pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk)
                umma_bf16_pair_if(issue, d, da + kk * (2048 / 16), db + kk * (2048 / 16), idesc, kk == 0 ? onto : 1u);
            } else {
              if (is_cut(left)) {
                if (!__all_sync(0xFFFFFFFFu, mbar_wait_cluster(&zeroed[s], (zph >> s) & 1, g.err, kErrMmaWait))) { ok = false; break; }
                zph ^= 1u << s;
              }
              tc_fence_after();
              for (int kk = 0; kk * 16 < left; ++kk)
                umma_bf16_pair_if(issue, d, da + kk * (2048 / 16), db + kk * (2048 / 16), idesc, kk == 0 ? onto : 1u);
            }
            umma_commit_pair_if(issue, bar0 + s * 8);
            umma_commit_pair_if(issue, bar1 + s * 8);
            if (++s == kWStages) { s = 0; ph ^= 1; }
            onto = 1;
            left -= kBK;
          }
          if (!ok) break;
          umma_commit_pair_if(issue, done0 + a * 8);
          umma_commit_pair_if(issue, done1 + a * 8);
          ++i;
        }
      }
    }
  } else if (warp == 2) {
    int s = 0;  // stage of the next block
    uint32_t cph = 0;
    for (int t = pair; t < tiles; t += pairs) {
      const int e = t / per_group;
      const int size = l.row[e + 1] - l.row[e], blocks = l.tile[e + 1] - l.tile[e];
      if (blocks == 0) continue;
      const int last = (s + blocks - 1) % kWStages;
      s = (s + blocks) % kWStages;
      const int valid = valid_rows(size, blocks - 1);
      if (!is_cut(valid)) continue;
      if (!__all_sync(0xFFFFFFFFu, mbar_wait(&cut[last], (cph >> last) & 1, g.err, kErrMmaWait))) break;
      cph ^= 1u << last;
      // MN-major chunks are rows of 128 bytes; both operands are zeroed (0 * inf is not 0)
      const int bytes = (((valid + 15) & ~15) - valid) * 128;
      uint8_t* stage = smem + last * S::kStageBytes + valid * 128;
      #pragma unroll 1
      for (int c = 0; c < 4; ++c)
        for (int b = lane * 16; b < bytes; b += 512)
          *reinterpret_cast<uint4*>(stage + c * S::kChunkBytes + b) = make_uint4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(mapa_shared(&zeroed[last], 0));
    }
  } else {
    const int q = warp & 3;           // TMEM lane quarter this warp may access
    const int half = (warp - 3) >> 2;  // columns 128 * half .. + 127 of the tile
    uint8_t* buf = staging + (warp - 3) * S::kOutBytes;
    const uint32_t acc_empty_leader0 = mapa_shared(&acc_empty[0], 0);
    const uint32_t acc_empty_leader1 = mapa_shared(&acc_empty[1], 0);
    int i = 0;
    bool ok = true;
    // This warp's part of tile t, brought into L2 ahead of the additions to it: a tile of one
    // accumulator during the tile before it, a longer one during its last accumulator.
    auto prefetch = [&](int t, bool ahead) {
      if (t >= tiles) return;
      const int e = t / per_group;
      const int blocks = l.tile[e + 1] - l.tile[e];
      if (blocks == 0 || ahead != (blocks <= kWChunk)) return;
      int tm, tn;
      wgrad_coords(t - e * per_group, blocks, tiles_m, tiles_n, tm, tn);
      const int row0 = tm * 256 + int(cta) * 128 + q * 32, col0 = tn * 256 + half * 128 + lane * 32;
      if (lane < 4 && row0 < g.n && col0 < g.k) tma_prefetch_3d_f32(&tma_c, col0, row0, e, g.err);
    };
    if (ACC) prefetch(pair, true);
    for (int t = pair; t < tiles && ok; t += pairs) {
      const int e = t / per_group;
      const int blocks = l.tile[e + 1] - l.tile[e];
      if (ACC) prefetch(t + pairs, true);
      if (blocks == 0 && ACC) continue;
      float acc[128];
      #pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.f;
      for (int c = 0; c < blocks; c += kWChunk, ++i) {
        const int a = i & 1;
        if (ACC && c + kWChunk >= blocks) prefetch(t, false);
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(&acc_full[a], (i >> 1) & 1, g.err, kErrEpiWait))) { ok = false; break; }
        tc_fence_after();
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t v[16];
          tmem_ld16(tmem_base + a * 256 + half * 128 + j * 16 + (uint32_t(q * 32) << 16), v);
          tmem_wait_ld();
          #pragma unroll
          for (int x = 0; x < 16; ++x) acc[j * 16 + x] += __uint_as_float(v[x]);
        }
        // Relaxed: this lane's bulk stores of the last tile are still under way, and a release
        // waits for them (1500 to 2400 cycles per tile; 64 groups of 94 rows, 1024 x 1416, written
        // 83 us against 93). In the row products, whose stores are smaller, it made no difference.
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote_tmem(a == 0 ? acc_empty_leader0 : acc_empty_leader1);
      }
      if (!ok) break;
      int tm, tn;
      wgrad_coords(t - e * per_group, blocks, tiles_m, tiles_n, tm, tn);
      const int row0 = tm * 256 + int(cta) * 128 + q * 32, col0 = tn * 256 + half * 128;
      if (row0 >= g.n) continue;
      constexpr int kCols = BF16 ? 64 : 32;  // of a 128-byte row of staging
      #pragma unroll
      for (int j = 0; j < 128; j += kCols) {
        if (col0 + j < g.k) {
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
          #pragma unroll
          for (int x = 0; x < 8; ++x) {  // the map's 128-byte swizzle: 16-byte unit x of row r is at x ^ r % 8
            uint8_t* unit = buf + lane * 128 + ((x ^ (lane & 7)) << 4);
            if (BF16) {
              const float* v = acc + j + 8 * x;  // the one rounding of the sum
              *reinterpret_cast<uint4*>(unit) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]),
                                                           pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
            } else {
              const float* v = acc + j + 4 * x;
              *reinterpret_cast<float4*>(unit) = make_float4(v[0], v[1], v[2], v[3]);
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            if (ACC) tma_add_3d_f32(&tma_c, buf, col0 + j, row0, e, g.err);
            else tma_store_3d(&tma_c, buf, col0 + j, row0, e, BF16 ? 8 : 4, g.err);
            bulk_commit();
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  cluster_sync();  // no CTA leaves while its pair may still touch its barriers or TMEM
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, S::kTmemCols);
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

// ``kernel`` on min(tiles, the pairs that can be resident at once) CTA pairs: a persistent grid
// larger than that would only queue. ``resident``: that number by device, 0 before it is known.
template <typename Kernel, typename... A>
void launch_pairs(Kernel kernel, int (&resident)[64], int threads, int smem, int64_t tiles, cudaStream_t st,
                  const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernel starts with pdl_enter()
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(unsigned(threads), 1, 1);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int dev = 0;
  RESIHP_CUDA_CHECK(cudaGetDevice(&dev));
  if (resident[dev] == 0) {
    RESIHP_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cfg.gridDim = dim3(2, 1, 1);
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = num_sms() / 2;
    }
    resident[dev] = n;
  }
  cfg.gridDim = dim3(2 * unsigned(std::min<int64_t>(tiles, resident[dev])), 1, 1);
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  RESIHP_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
}

template <int TN, bool W_MN>
void launch_rows(int64_t tiles, const CUtensorMap& tw, const CUtensorMap& ta, const Args& g, cudaStream_t st) {
  static int resident[64] = {0};
  launch_pairs(grouped_rows_kernel<TN, W_MN>, resident, 192, RowTile<TN>::kSmem, tiles, st, tw, ta, g);
}

template <bool ACC, bool BF16>
void launch_wgrad(int64_t tiles, const CUtensorMap& tdy, const CUtensorMap& tx, const CUtensorMap& tc, const Args& g,
                  cudaStream_t st) {
  static int resident[64] = {0};
  launch_pairs(grouped_wgrad_kernel<ACC, BF16>, resident, kWThreads, WgradTile::kSmem, tiles, st, tdy, tx, tc, g);
}

template <int TN>
void launch_rows_tn(const void* a, int64_t lda, const void* w, int64_t ldw, int64_t w_group, bool w_mn,
                    const GroupedShape& s, const Args& g, cudaStream_t st) {
  const int64_t tiles_f = (s.n + 255) / 256;
  const int64_t most = (int64_t(s.rows) + TN - 1) / TN + s.groups + 1;  // row tiles, if every group cuts one
  RESIHP_CHECK(most * tiles_f <= INT32_MAX, "grouped products: too many tiles");
  const CUtensorMap ta = make_tma_2d_bf16(a, s.rows, s.k, lda, 64, TN / 2);
  const CUtensorMap tw = w_mn ? make_tma_3d_bf16(w, s.groups, s.k, s.n, ldw, w_group, 64, 64)
                              : make_tma_3d_bf16(w, s.groups, s.n, s.k, ldw, w_group, 64, 128);
  if (w_mn) launch_rows<TN, true>(most * tiles_f, tw, ta, g, st);
  else launch_rows<TN, false>(most * tiles_f, tw, ta, g, st);
}

void check_shape(const GroupedShape& s) {
  RESIHP_CHECK(s.groups >= 1 && s.groups <= kMaxGroups, "grouped products take 1 to ", kMaxGroups, " groups");
  RESIHP_CHECK(s.n >= 8 && s.k >= 8 && s.n % 8 == 0 && s.k % 8 == 0,
               "grouped products need widths that are multiples of 8 (16-byte vectors)");
  RESIHP_CHECK(s.rows >= 0, "grouped products: negative row count");
}

}  // namespace

bool grouped_paces(const GroupedShape& s) {
  return s.k >= kPaceDepth && int64_t(s.rows / 256) * ((s.n + 255) / 256) >= num_sms();
}

void grouped_rows(const void* a, int64_t lda, const void* w, int64_t ldw, int64_t w_group, bool w_mn, void* c,
                  int64_t ldc, const GroupedShape& s, unsigned* pace, int* err, cudaStream_t st) {
  check_shape(s);
  if (s.rows == 0) return;
  if (pace != nullptr) RESIHP_CUDA_CHECK(cudaMemsetAsync(pace, 0, sizeof(unsigned), st));
  RESIHP_CHECK(reinterpret_cast<uintptr_t>(c) % 16 == 0 && ldc % 8 == 0, "grouped output must be 16-byte aligned");
  const Args g{c, ldc, s.offsets, s.groups, s.rows, s.n, s.k, pace, err};
  // Few rows per group: the weights' bytes set the time, and narrow row tiles leave room for
  // eight of their stages in flight instead of six. At 100 rows a group (eight groups, 2048 >
  // 11008) 64.3 against 66.7 us, at 94 uneven ones (64 groups, 1024 > 1416) 44.3 against 46.9;
  // at 150 uneven ones 73.7 against 70.6: groups of more than 128 rows read their weights twice.
  // The average is all the host knows: how uneven the groups are stands on the device.
  if (s.rows <= int64_t(112) * s.groups) launch_rows_tn<128>(a, lda, w, ldw, w_group, w_mn, s, g, st);
  else launch_rows_tn<256>(a, lda, w, ldw, w_group, w_mn, s, g, st);
}

void grouped_wgrad(const void* dy, int64_t lddy, const void* x, int64_t ldx, void* c, bool bf16, bool accumulate,
                   const GroupedShape& s, int* err, cudaStream_t st) {
  check_shape(s);
  RESIHP_CHECK(reinterpret_cast<uintptr_t>(c) % 16 == 0, "grouped weight gradient must be 16-byte aligned");
  RESIHP_CHECK(!bf16 || !accumulate, "grouped weight gradient: only fp32 is accumulated into");
  if (s.rows == 0) {
    if (!accumulate) RESIHP_CUDA_CHECK(cudaMemsetAsync(c, 0, (bf16 ? 2 : 4) * size_t(s.groups) * s.n * s.k, st));
    return;
  }
  const int64_t tiles = int64_t(s.groups) * ((s.n + 255) / 256) * ((s.k + 255) / 256);
  RESIHP_CHECK(tiles <= INT32_MAX, "grouped products: too many tiles");
  const CUtensorMap tdy = make_tma_2d_bf16(dy, s.rows, s.n, lddy, 64, kBK);
  const CUtensorMap tx = make_tma_2d_bf16(x, s.rows, s.k, ldx, 64, kBK);
  const CUtensorMap tc = bf16 ? make_tma_3d_bf16(c, s.groups, s.n, s.k, s.k, int64_t(s.n) * s.k, 64, 32)
                              : make_tma_3d_f32(c, s.groups, s.n, s.k, 32);
  const Args g{c, 0, s.offsets, s.groups, s.rows, s.n, s.k, nullptr, err};
  if (accumulate) launch_wgrad<true, false>(tiles, tdy, tx, tc, g, st);
  else if (bf16) launch_wgrad<false, true>(tiles, tdy, tx, tc, g, st);
  else launch_wgrad<false, false>(tiles, tdy, tx, tc, g, st);
}

}  // namespace resihp
