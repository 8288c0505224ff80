// Products whose weight is picked by the row, for sm_100a:
//
//   C[r, :] = act(A[r, :] * B[e] + bias[e])   for off[e] <= r < off[e + 1]
//
// A is T x K (rows sorted by group), B a stack of E weights K x N (or stored
// N x K), 16-bit inputs (fp16 or bf16), fp32 accumulation, one rounding to
// the inputs' type.  The counts of the groups are only known on the device:
// every CTA reads the offsets, lays the groups' tiles out one after the other
// (a prefix sum in shared memory) and walks its share, so nothing is
// synchronised with the host and one launch serves any split of the rows.
//
// The weights sit on the 128 TMEM lanes (MMA M) and the rows are the MMA N,
// i.e. a tile computes C^T = B^T A^T.  Row counts are ragged and the MMA N is
// a run-time field with steps of 16 (32 for a CTA pair), so a group of 37 rows costs 48
// rows of MMA work and of A traffic; with the rows on the lanes it would cost
// 128 (256).  A group's rows are cut into equal tiles of at most TM rows.
//
//   CG = 2, TM = 256: a CTA pair owns 256 columns x up to 256 rows; each CTA
//     loads its 128 columns of B and half of the rows (no multicast).  What
//     bounds it is the way from L2 (10 TB/s over the machine) and the power cap.
//   CG = 2, TM = 512: two such tiles one below the other share the K blocks of
//     B: 48 KiB per stage and CTA instead of twice 32.  Each has an accumulator
//     of its own, so the next tile starts on one while the other is read out.
//   CG = 1, TM = 64: a CTA owns 128 columns x up to 64 rows; a short last wave
//     is split along K over the 2, 4 or 8 CTAs of a cluster.  The ring holds
//     over 100 KiB of weights in flight.  For groups of few rows, whose cost is reading the weights
//     (steady state 7.3 TB/s on weights stored K x N, 6.2 stored N x K), and
//     for problems too small to fill the machine with pair tiles.  The
//     partial sums cross through distributed shared memory by bulk copies: CTA r
//     finishes every cluster's r-th part of the rows, summing in CTA order.
//     (Pieces through global memory with a ticket were measured first: joining
//     two of them cost 3 us, four times this path.)
//
// Roles: warps 0 and 10 are the TMA producers of the weights and of the rows (one
// thread issues a load in 100-150 cycles, so two share them), warp 1 owns TMEM
// and issues the MMAs, warps 2..9 are the epilogue, in two groups that take
// alternate chunks of rows.  The accumulator holds C transposed:
// a thread owns one column of C and walks the rows, so bias is one value per
// thread, and the 32-row chunks go through shared memory to become rows of
// 256 bytes.  A chunk that lies wholly inside its group is stored by TMA, a
// cut one row by row: the rows behind it are the next group's.  Rows that the
// last A box of a group reads past the group's end only reach accumulator
// columns that are not stored, so nothing in them (inf, NaN) can spread.
//
// LORA = true adds low-rank adapters picked by the row to one shared product
// (E = 1, no offsets):  C[r, :] = act(A[r, :] * B + h[r, :] * up[a_r] + bias).
// h (fp32, scaled) comes from lora_shrink (gemm_lora_kernel.cuh), which runs
// beside this kernel's first K blocks: only the rows of h wait for it.  The
// epilogue warps list the distinct adapters of a tile's rows while its K
// blocks are multiplied.  After the K blocks of a tile come its
// adapter blocks, 32 ranks of one adapter each, which pass through the same
// ring: the weight slot of a stage holds `up` (64 ranks wide as TMA's swizzle
// wants it, of which 32 are used), and its row slot is filled by the epilogue
// warps: row r holds h[r] when the row picked this adapter and zeros when not,
// so rows with different adapters share a tile.  h is split into two bf16
// numbers, h = hi + lo with |lo| <= half a step of hi, side by side in the 64
// columns of the slot, each multiplied with the same `up`: what tensor cores
// take is 16-bit, and rounding h to one would cost as much accuracy as the
// result's own rounding does.  bf16 for fp16 operands too, since h is an fp32
// number of any size (a small `scale` with a large `up`, or the other way
// round): two fp16 parts end at 65504 and keep ever fewer bits below 2^-9.  Both
// operands of an MMA are of one type, so an fp16 `up` is split likewise, into
// two bf16 numbers that add up to it exactly, in the ranks of its slot that are
// not used: four products to a rank instead of two, and the epilogue warps, which
// read every landed tile anyway (see below), write it back (64 rows, 32 adapters
// of rank 16, 4096 x 4096: 19.4 us, 18.9 with fp16 parts).
//
// A row that did not pick the adapter multiplies `up` with zeros, and 0 * inf
// is not 0; nor is hi * inf + lo * inf the h * inf of a row that did (lo may be
// 0 or have the other sign).  So the thread that owns a column looks its ranks
// over once they have landed, replaces an inf or NaN by 0 in shared memory, and
// adds what it replaced to the rows of that adapter in the epilogue: one
// request's weights cannot reach another's rows, and what its own rows get does
// not depend on its neighbours.
#pragma once
#include "gemm_lora_kernel.cuh"
#include "gemm_sm100_kernel.cuh"

namespace idb {

constexpr int kGrpCols = 128;      // columns of C per CTA: the TMEM lanes
constexpr int kMaxGroups = 1024;   // bounded by the offset tables in shared memory
constexpr int kGrpChunk = 32;      // rows of C per epilogue step
constexpr int kGrpRaster = 8;      // tiles of rows walked before the next column tile

// A's rows come in one box per K block, the smallest that holds a CTA's share
// of the tile's rows.  A full pair tile draws 64 bytes per clock and SM from
// L2, which is what the SM's port gives (measured: 60 without the MMAs), so
// rows that are not needed cost time.
constexpr int kBoxes = 6;
__host__ __device__ constexpr int box_rows(int tm, int i) {   // 128, 112, 96, 80, 64, 32, or 64, 48, 32, 16
  return tm >= 256 ? (i < 5 ? 128 - 16 * i : 32) : 64 - 16 * i;
}
__host__ __device__ constexpr int box_count(int tm) { return tm >= 256 ? 6 : 4; }

struct alignas(64) GroupedMaps {
  CUtensorMap a[kBoxes];
  CUtensorMap b, c, u;
};

struct GroupedParams {
  const void* offsets;  // int32 or int64 [E + 1]; null: one group of all T rows
  int off64;
  int E;
  int T, N, K;
  int kb_total;      // ceil(K / 64)
  int tiles_n;       // ceil(N / (128 * CG))
  int first_box;     // the largest box of A that T rows can need
  int b_kmaj;        // B[e] stored N x K
  int b_wide;        // stored K x N with N a multiple of 64: both 64-column atoms in one box
  int bf16;
  int act;
  const unsigned short* bias;  // [E, N] or null
  unsigned short* C;
  long long ldc;
  int c_tma;         // C is TMA-addressable
  int c_vec;         // C rows are 16-byte aligned
  int zero_rest;     // rows outside [off[0], off[E]): 1 written as 0, 0 left as they are
  int* err;
  // LORA
  const float* h;    // [T, h_pitch]
  int h_pitch;
  int L, R;
  const void* adapter;
  int adapter64;
  int up_kmaj;       // up[a] stored N x R
  int up_wide;
  const unsigned short* up;
  long long ld_up, stride_up;
  int packed;        // an operand is a copy made by this call
};

constexpr int kLoraRanks = 32;   // ranks per adapter block

// Two groups of four epilogue warps (one warp per TMEM lane quarter each): they
// take alternate chunks of rows, and alternate adapter blocks.
constexpr int kGrpEpiWarps = 8;
constexpr int kGrpThreads = 64 + 32 * kGrpEpiWarps + 32;
constexpr int kGrpRowsWarp = 2 + kGrpEpiWarps;   // producer of the rows; warp 0 produces the weights

template <int CG, int TM, int STAGES, bool LORA>
struct GroupedPlan {
  static constexpr int kStep = 16 * CG;                  // granularity of a tile's rows (MMA N)
  static constexpr int kSubs = TM > 256 ? 2 : 1;         // parts of a tile's rows, each an accumulator of its own
  static constexpr int kSubRows = TM / kSubs;
  static constexpr int kTokRows = TM / CG;               // rows of A held by this CTA
  static constexpr int kSubBytes = kSubRows / CG * kBK * 2;   // rows of one part
  static constexpr int kWBytes = kGrpCols * kBK * 2;     // 16 KiB of B
  static constexpr int kTBytes = kTokRows * kBK * 2;
  static constexpr int kStageBytes = kWBytes + kTBytes;
  static constexpr int kOutBytes = kGrpChunk * kGrpCols * 2;  // staging of one chunk
  static constexpr int kOffW = 0;
  static constexpr int kOffT = kOffW + STAGES * kWBytes;
  static constexpr int kOffOut = kOffT + STAGES * kTBytes;
  static constexpr int kOffRx = kOffOut + 2 * kOutBytes;  // fp32 sums from the cluster
  static constexpr int kOffBar = kOffRx + (CG == 1 ? TM * kGrpCols * 4 : 0);
  // full, empty, land, built, tmem_full[2], tmem_empty[2], rx_full, list, list_read, done
  static constexpr int kNumBars = 4 * STAGES + 8;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kOffScan = kOffMisc + 32;         // warp totals
  static constexpr int kOffRows = (kOffScan + 64 + 15) / 16 * 16;   // group starts [E + 1]
  static constexpr int kOffTiles = kOffRows + (kMaxGroups + 1) * 4;  // first tile of each group [E + 1]
  static constexpr int kUsed = kOffTiles + (kMaxGroups + 1) * 4;
  static constexpr int kDynamicBytes = kUsed + 1024;
  static constexpr uint32_t kTmemCols = 2 * kSubRows;    // two accumulators
  static_assert(TM % (32 * CG) == 0 && kSubRows <= 256 && kSubs * kSubRows == TM, "rows of a tile");
  static_assert(kTBytes % 1024 == 0 && kOffOut % 1024 == 0, "swizzled tiles need 1024-byte alignment");
  static_assert(kDynamicBytes <= 227 * 1024, "shared memory of one CTA");
};

// offsets[i], kept inside [0, T].
__device__ __forceinline__ int group_offset(const void* offsets, int off64, int i, int T, bool& bad) {
  const long long v = off64 ? static_cast<const long long*>(offsets)[i] : static_cast<const int*>(offsets)[i];
  bad |= v < 0 || v > T;
  return static_cast<int>(v < 0 ? 0 : (v > T ? T : v));
}

// Row tiles of a group of n rows: `count` tiles of `rows` rows each (the last
// one may be shorter), rows a multiple of STEP and at most TM.  Equal tiles
// rather than full ones and a rest: the same count with less padding.
template <int TM, int STEP>
__host__ __device__ __forceinline__ void row_tiles(int n, int& count, int& rows) {
  count = (n + TM - 1) / TM;
  rows = (count > 1 ? (n + count - 1) / count + STEP - 1 : n + STEP - 1) / STEP * STEP;
}

// Few groups: every warp makes the same tables for itself (all write the same
// values), so no warp waits for another.  A lane owns up to 8 consecutive
// groups, its offsets in flight at once.  False if the offsets are bad.
constexpr int kWarpScanGroups = 256;
template <class Units>
__device__ __forceinline__ bool scan_groups_warp(const void* offsets, int off64, int E, int T, int* rows, int* first,
                                                 Units units) {
  constexpr int kMost = kWarpScanGroups / 32;
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int per = (E + 31) >> 5, g0 = lane * per;
  int v[kMost + 1];
  bool bad = false;
#pragma unroll
  for (int j = 0; j <= kMost; ++j) {
    if (j <= per) v[j] = group_offset(offsets, off64, min(g0 + j, E), T, bad);
  }
  int sum = 0;
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    if (j < per) {
      bad |= v[j + 1] < v[j];
      sum += units(v[j + 1] - v[j]);   // 0 past the last group
    }
  }
  int run = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, run, d);
    if (lane >= d) run += up;
  }
  int base = run - sum;
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    if (j < per && g0 + j < E) {
      rows[g0 + j] = v[j];
      first[g0 + j] = base;
      base += units(v[j + 1] - v[j]);
      if (g0 + j == E - 1) {
        rows[E] = v[j + 1];
        first[E] = base;
      }
    }
  }
  __syncwarp();
  return __all_sync(0xffffffffu, !bad) != 0;
}

// Fills rows[0..E] with the group starts and first[0..E] with an exclusive
// prefix sum of units(rows of the group); first[E] is the total.  Called by
// all NT threads of the CTA.  Offsets that decrease or leave [0, T] set the
// error bit and are read as the nearest valid ones (a running maximum), so
// that no group ever owns another's rows.
template <int NT, class Units>
__device__ __forceinline__ void scan_groups(const void* offsets, int off64, int E, int T, int* rows, int* first,
                                            int* scratch, int* err, Units units) {
  const int tid = static_cast<int>(threadIdx.x);
  if (offsets == nullptr) {   // one group
    if (tid == 0) {
      rows[0] = 0;
      rows[1] = T;
      first[0] = 0;
      first[1] = units(T);
    }
    __syncthreads();
    return;
  }
  bool bad = false;
  for (int i = tid; i <= E; i += NT) rows[i] = group_offset(offsets, off64, i, T, bad);
  __syncthreads();
  // each thread owns a run of consecutive groups
  const int per = (E + NT - 1) / NT;
  const int g0 = min(E, tid * per), g1 = min(E, g0 + per);
  int sum = 0, run = 0;
  auto scan = [&] {
    sum = 0;
    for (int g = g0; g < g1; ++g) {
      bad |= rows[g + 1] < rows[g];
      sum += units(rows[g + 1] - rows[g]);
    }
    run = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, run, d);
      if ((tid & 31) >= d) run += up;
    }
    if ((tid & 31) == 31) scratch[tid >> 5] = run;
  };
  scan();
  if (__syncthreads_or(bad ? 1 : 0)) {
    if (tid == 0) {
      for (int i = 0; i < E; ++i) rows[i + 1] = max(rows[i + 1], rows[i]);
      atomicOr(err, kDevErrBadOffsets);
    }
    __syncthreads();
    scan();
    __syncthreads();
  }
  int base = run - sum;
  for (int w = 0; w < (tid >> 5); ++w) base += scratch[w];
  for (int g = g0; g < g1; ++g) {
    first[g] = base;
    base += units(rows[g + 1] - rows[g]);
  }
  if (tid == NT - 1) first[E] = base;   // the last thread's base ends at the total
  __syncthreads();
}

// The group whose units hold unit u: the last g with first[g] <= u.
__device__ __forceinline__ int find_group(const int* first, int E, int u) {
  int lo = 0, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The tiles of one CTA (pair): whole ones, `stride` apart, and then perhaps a
// share of the last, short wave's.
//  * Single CTAs: a last wave with no more tiles than clusters is split along
//    K over the CTAs of each cluster; it takes half the time with clusters of
//    two (32 rows over 64 experts, 200 tiles on 148 CTAs: the 52 of the second
//    wave).
//  * Pairs with tiles of two parts: a last wave that half of the pairs could do
//    is done part by part by all of them.
struct GroupedWalk {
  int t, stride;
  int whole;       // tiles that are walked whole
  int split_tile;  // the one to split along K; at or past `tiles`: none
  int tiles;
  int part;        // the only part of the tile that next() gave, or -1

  template <int SUBS>
  __device__ __forceinline__ bool next(int& tile, bool& split) {
    if (SUBS == 2) {
      const int i = t - whole;
      part = i < 0 ? -1 : i & 1;
      tile = i < 0 ? t : whole + (i >> 1);
      t += stride;
      return tile < tiles;
    }
    split = t >= whole;
    tile = split ? split_tile : t;
    if (split) split_tile = tiles;
    t += split ? 0 : stride;
    return tile < tiles;
  }
};

template <int CG, int SUBS>
__device__ __forceinline__ GroupedWalk grouped_walk(int tiles, int cta, int ctas, int worker, int workers) {
  if (CG == 2) {
    const int waves = tiles / workers, rest = tiles - waves * workers;
    return {worker, workers, SUBS == 2 && 2 * rest <= workers ? waves * workers : tiles, tiles, tiles, -1};
  }
  const int waves = tiles / ctas, rest = tiles - waves * ctas;
  const int whole = rest <= workers ? waves * ctas : tiles;
  return {cta, ctas, whole, whole + worker, tiles, -1};
}

struct GroupedUnit {
  int e;      // group
  int rt;     // row tile of the group
  int tn;     // column tile
  int row0;   // first row of A and C
  int rows;   // rows of C to store
  int nmma;   // MMA N: rows rounded up
  int subs;   // parts of the rows; `rows` and `nmma` are those of the first
  int rest;   // rows of the second

  // Moves on to the second part.
  template <int STEP>
  __device__ __forceinline__ void second() {
    row0 += rows;
    rows = rest;
    nmma = (rest + STEP - 1) / STEP * STEP;
  }
};

template <int CG, int TM>
__device__ __forceinline__ GroupedUnit grouped_unit(const GroupedParams& p, const int* rows, const int* first, int t,
                                                    int part) {
  GroupedUnit u;
  u.e = find_group(first, p.E, t);
  int count, tr;
  row_tiles<TM, 16 * CG>(rows[u.e + 1] - rows[u.e], count, tr);
  const int local = t - first[u.e];
  if (count == 1) {   // no divisions on the way to the first load
    u.tn = local;
    u.rt = 0;
  } else {
    // 4096 rows at a time for pairs: 4096 rows, 4096 x 14336 in 256-row tiles 443
    // us, 451 by 2048 rows; 8192 rows, 14336 x 4096 in 512-row tiles 739 us, 762
    // by 8192 rows
    constexpr int kRaster = CG == 2 ? 4096 / TM : kGrpRaster;
    const int per = kRaster * p.tiles_n;
    const int g = local / per;
    const int gs = min(count - g * kRaster, kRaster);
    const int r = local - g * per;
    u.tn = r / gs;
    u.rt = g * kRaster + r % gs;
  }
  u.row0 = rows[u.e] + u.rt * tr;
  u.rows = min(tr, rows[u.e + 1] - u.row0);
  u.subs = 1;
  u.rest = 0;
  if (TM > 256 && u.rows > 256) {
    const int half = ((u.rows + 1) / 2 + 31) / 32 * 32;
    u.subs = 2;
    u.rest = u.rows - half;
    u.rows = half;
  }
  if (TM > 256 && part >= 0) {   // one part only, which may have no rows
    if (part == 1) u.row0 += u.rows, u.rows = u.rest;
    u.subs = 1;
    u.rest = 0;
  }
  u.nmma = (u.rows + 16 * CG - 1) / (16 * CG) * (16 * CG);
  return u;
}

// Rows outside every group, written as zeros by the epilogue warps of the grid.
__device__ __forceinline__ void zero_rows(const GroupedParams& p, int lo, int hi, int thread, int threads) {
  const int outside = lo + (p.T - hi);
  for (int i = static_cast<int>(blockIdx.x); i < outside; i += static_cast<int>(gridDim.x)) {
    unsigned short* row = p.C + static_cast<long long>(i < lo ? i : hi + (i - lo)) * p.ldc;
    int c = 0;
    if (p.c_vec) {
      for (c = thread * 8; c + 8 <= p.N; c += threads * 8) {
        *reinterpret_cast<uint4*>(row + c) = make_uint4(0u, 0u, 0u, 0u);
      }
      c = p.N / 8 * 8 + thread;
    } else {
      c = thread;
    }
    for (; c < p.N; c += threads) row[c] = 0;
  }
}

__device__ __forceinline__ bool nonfinite16(uint32_t h, bool bf16) {
  const uint32_t exponent = bf16 ? 0x7F80u : 0x7C00u;
  return (h & exponent) == exponent;
}

// The same for both halves of a word: bits 15 and 31 say which.  An exponent
// of all ones plus one in its lowest place carries into the sign bit's place.
__device__ __forceinline__ uint32_t nonfinite_pair(uint32_t w, bool bf16) {
  return ((w & (bf16 ? 0x7F807F80u : 0x7C007C00u)) + (bf16 ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}

// RANKS ranks of one row as 16-byte chunks of bf16: hi in the first half of them,
// lo in the second.  hi + lo is h to 2^-16 of it.
template <int RANKS>
__device__ __forceinline__ void split_ranks(const float* h, int valid, uint4 (&out)[RANKS / 4]) {
  uint32_t hi[RANKS / 2], lo[RANKS / 2];
  uint32_t seen = 0;
#pragma unroll
  for (int i = 0; i < RANKS; i += 4) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < valid) v = __ldcg(reinterpret_cast<const float4*>(h + i));   // the pitch of h is a multiple of 16 ranks
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x = e ? v.z : v.x, y = e ? v.w : v.y;
      const uint32_t top = pack_16bit(x, y, true);
      hi[i / 2 + e] = top;
      lo[i / 2 + e] = pack_16bit(x - __uint_as_float(top << 16), y - __uint_as_float(top & 0xFFFF0000u), true);
      seen |= nonfinite_pair(top, true);
    }
  }
  // An infinite h is infinite in hi, and lo must not undo that (inf - inf); a
  // NaN stays in hi too.  A finite h that rounds to infinity has the largest
  // finite hi.
  if (seen) {
#pragma unroll
    for (int i = 0; i < RANKS / 2; ++i) {
      const uint32_t bad = nonfinite_pair(hi[i], true);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (!(bad & (e ? 0x80000000u : 0x8000u))) continue;
        const uint32_t keep = e ? 0x0000FFFFu : 0xFFFF0000u;
        const float x = __ldcg(h + 2 * i + e);
        uint32_t rest = 0;
        if (fabsf(x) < __int_as_float(0x7F800000)) {
          const uint32_t top = (__float_as_uint(x) & 0x80000000u) | 0x7F7F0000u;
          hi[i] = (hi[i] & keep) | (e ? top : top >> 16);
          rest = to_16bit(x - __uint_as_float(top), true);
        }
        lo[i] = (lo[i] & keep) | (rest << (16 * e));
      }
    }
  }
#pragma unroll
  for (int c = 0; c < RANKS / 8; ++c) {
    out[c] = make_uint4(hi[4 * c], hi[4 * c + 1], hi[4 * c + 2], hi[4 * c + 3]);
    out[RANKS / 8 + c] = make_uint4(lo[4 * c], lo[4 * c + 1], lo[4 * c + 2], lo[4 * c + 3]);
  }
}

// Two fp16 numbers f as two pairs of bf16 numbers, top + rest = f exactly: top is
// 15/16 f cut to 8 bits, and what is left of f's 11 bits fits into 8 (the first of
// them 3 or 4 places below f's).  Neither is 0 nor has the other sign unless f is
// 0, so that an infinite h times both adds up to what h * f is.
__device__ __forceinline__ void split_up(uint32_t f, uint32_t& top, uint32_t& rest) {
  const float x = from_16bit(static_cast<unsigned short>(f), false);
  const float y = from_16bit(static_cast<unsigned short>(f >> 16), false);
  const uint32_t a = __float_as_uint(0.9375f * x), b = __float_as_uint(0.9375f * y);
  top = __byte_perm(a, b, 0x7632);
  rest = __byte_perm(__float_as_uint(x - __uint_as_float(a & 0xFFFF0000u)),
                     __float_as_uint(y - __uint_as_float(b & 0xFFFF0000u)), 0x7632);
}

// Makes the first 16 `steps` ranks of a landed `up` tile an operand of the
// adapter's MMAs: inf and NaN become zeros, and fp16 numbers are split, the
// rests 32 ranks on.  Says whether this thread found an inf or NaN.  128
// threads, two 16-byte chunks each per 16 ranks: a tile stored N x R has them in
// row `thread`, one stored R x N in rows 0..15 (16..31) of both atoms.
__device__ __forceinline__ bool prepare_up(uint8_t* tile, int thread, int steps, bool kmaj, bool bf16) {
  uint32_t seen = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= 2 * steps) break;
    uint4* at = reinterpret_cast<uint4*>(kmaj ? tile + thread * 128 + ((i ^ (thread & 7)) << 4)
                                              : tile + (i & 1) * (kBK * 128) + ((i >> 1) * 128 + thread) * 16);
    uint4 v = *at;
    const uint32_t bad = nonfinite_pair(v.x, bf16) | nonfinite_pair(v.y, bf16) | nonfinite_pair(v.z, bf16) |
                         nonfinite_pair(v.w, bf16);
    if (bad) {
      auto cleared = [&](uint32_t w) { return w & ~((nonfinite_pair(w, bf16) >> 15) * 0xFFFFu); };
      v = make_uint4(cleared(v.x), cleared(v.y), cleared(v.z), cleared(v.w));
      seen = 1;
    }
    if (!bf16) {
      uint4 rest;
      split_up(v.x, v.x, rest.x);
      split_up(v.y, v.y, rest.y);
      split_up(v.z, v.z, rest.z);
      split_up(v.w, v.w, rest.w);
      // 32 ranks on: four chunks of the row, or 32 rows (the swizzle repeats every 8)
      *reinterpret_cast<uint4*>(kmaj ? tile + thread * 128 + (((i + 4) ^ (thread & 7)) << 4)
                                     : reinterpret_cast<uint8_t*>(at) + kLoraRanks * 128) = rest;
    }
    if (bad || !bf16) *at = v;
  }
  return seen != 0;
}

// What prepare_up took out of row t's value in column n in the adapter
// blocks [b0, b1) of its tile.
__device__ __noinline__ float nonfinite_terms(const GroupedParams& p, const int* list, int adapters, int b0, int b1,
                                              int t, int n) {
  bool bad = false;
  const int a = adapter_of(p.adapter, p.adapter64, t, p.L, bad);
  int ai = 0;
  while (ai < adapters && list[ai] != a) ++ai;
  float sum = 0.0f;
  if (a < 0 || ai == adapters) return sum;
  for (int r = 0; r < p.R; ++r) {
    const int b = r / kLoraRanks * adapters + ai;
    if (b < b0 || b >= b1) continue;
    const unsigned short w = p.up[a * p.stride_up + (p.up_kmaj ? n * p.ld_up + r : r * p.ld_up + n)];
    if (nonfinite16(w, p.bf16 != 0)) {
      sum += p.h[static_cast<long long>(t) * p.h_pitch + r] * from_16bit(w, p.bf16 != 0);
    }
  }
  return sum;
}

// x * Phi(x), Phi the normal distribution, without the branches of the math
// library's error function (whose two paths kept the 32 values of a chunk from overlapping: the epilogue of a
// 256 x 256 tile took 42000 cycles, more than its mainloop at K = 4096).
//
// With a = |x| and q(a) = 1 - Phi(a) = erfc(a / sqrt 2) / 2:
//   x Phi(x) = max(x, 0) - a q(a)        (both signs of x)
//   q(a) = exp(-a^2 / 2) t Q(t),  t = 1 / (1 + 0.31 a)
// where Q is the polynomial of degree 7 with the least relative error to
// exp(a^2 / 2) q(a) / t over 0 <= a <= 20 (an iteratively reweighted
// least-squares fit in 64 bits), 1.7e-7.  In fp32 the result errs by at most
// 4 units of 2^-24 |x| and by 1.5e-6 of its value wherever fp16 is normal.
// x / 2 + |x| / 2 rather than max(x, 0), so that a NaN stays one (halves first:
// x + |x| overflows where bf16 does not).
__device__ __forceinline__ float gelu(float x) {
  const float a = fminf(fabsf(x), 20.0f);
  float t, e;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.31f, a, 1.0f)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(a * a * -0.72134752f));   // -log2(e) / 2
  float q = 0.035917483f;
  q = fmaf(q, t, -0.14193712f);
  q = fmaf(q, t, 0.15567426f);
  q = fmaf(q, t, -0.015496778f);
  q = fmaf(q, t, 0.11044533f);
  q = fmaf(q, t, 0.10766225f);
  q = fmaf(q, t, 0.12407906f);
  q = fmaf(q, t, 0.1236556f);
  return fmaf(-a, q * t * e, fmaf(0.5f, fabsf(x), 0.5f * x));
}

// gelu of two values with packed arithmetic, operation for operation the same.
__device__ __forceinline__ void gelu2(float& x0, float& x1) {
  const float a0 = fminf(fabsf(x0), 20.0f), a1 = fminf(fabsf(x1), 20.0f);
  const uint64_t a = pack_f32x2(a0, a1);
  const uint64_t d = fma_f32x2(pack_f32x2(0.31f, 0.31f), a, pack_f32x2(1.0f, 1.0f));
  const uint64_t s = mul_f32x2(mul_f32x2(a, a), pack_f32x2(-0.72134752f, -0.72134752f));
  float d0, d1, s0, s1, t0, t1, e0, e1;
  unpack_f32x2(d, d0, d1);
  unpack_f32x2(s, s0, s1);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(d0));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(d1));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(s0));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(s1));
  const uint64_t t = pack_f32x2(t0, t1);
  uint64_t q = pack_f32x2(0.035917483f, 0.035917483f);
  q = fma_f32x2(q, t, pack_f32x2(-0.14193712f, -0.14193712f));
  q = fma_f32x2(q, t, pack_f32x2(0.15567426f, 0.15567426f));
  q = fma_f32x2(q, t, pack_f32x2(-0.015496778f, -0.015496778f));
  q = fma_f32x2(q, t, pack_f32x2(0.11044533f, 0.11044533f));
  q = fma_f32x2(q, t, pack_f32x2(0.10766225f, 0.10766225f));
  q = fma_f32x2(q, t, pack_f32x2(0.12407906f, 0.12407906f));
  q = fma_f32x2(q, t, pack_f32x2(0.1236556f, 0.1236556f));
  q = mul_f32x2(mul_f32x2(q, t), pack_f32x2(e0, e1));
  const uint64_t half = pack_f32x2(0.5f, 0.5f);
  const uint64_t r = fma_f32x2(half, pack_f32x2(fabsf(x0), fabsf(x1)), mul_f32x2(half, pack_f32x2(x0, x1)));
  unpack_f32x2(fma_f32x2(pack_f32x2(-a0, -a1), q, r), x0, x1);
}

// `count` staged rows (128 columns of 16 bits each) to C at row `row`, column
// n0, by `threads` threads.
__device__ __forceinline__ void store_rows(const GroupedParams& p, const uint8_t* buf, int row, int count, int n0,
                                           int thread, int threads) {
  unsigned short* crow = p.C + static_cast<long long>(row) * p.ldc + n0;
  if (p.c_vec) {
    const int seg = (thread & 15) * 8;
    const int valid = min(8, p.N - n0 - seg);   // columns of this thread's 16 bytes inside C
#pragma unroll 1
    for (int r = thread >> 4; r < count; r += threads >> 4) {
      const unsigned short* src = reinterpret_cast<const unsigned short*>(buf + r * (kGrpCols * 2)) + seg;
      unsigned short* out = crow + r * p.ldc + seg;
      if (valid == 8) {
        *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(src);
      } else {
        for (int c = 0; c < valid; ++c) out[c] = src[c];
      }
    }
  } else {
    const int c = thread & 127;
    if (n0 + c >= p.N) return;
#pragma unroll 4
    for (int r = thread >> 7; r < count; r += threads >> 7) {
      crow[r * p.ldc + c] = reinterpret_cast<const unsigned short*>(buf + r * (kGrpCols * 2))[c];
    }
  }
}

// Where the K blocks of 128 columns of a stacked weight lie in its tensor map.
//
// The number of TMA instructions per K block is what bounds a full pair tile
// if anything but the MMAs does: a thread issues one in 100-150 cycles, and
// six per block (four boxes of 32 rows of A, two 64-column atoms of B) took
// 830 cycles where the MMAs take 512.  So each operand comes in one box, the
// two atoms of a row-major weight through a map that sees the columns as
// (64, N / 64) where N allows it, and the two operands have a producer each.
struct WeightBoxes {
  int x, y, z, e;   // of the first K block
  int dx, dy;       // per K block
  bool two;         // a second box for the other atom
};

__device__ __forceinline__ WeightBoxes weight_boxes(bool kmaj, bool wide, int k0, int col, int e) {
  if (kmaj) return {k0, col, 0, e, kBK, 0, false};
  if (wide) return {0, k0, col >> 6, e, 0, kBK, false};
  return {col, k0, 0, e, 0, kBK, true};
}

template <bool PAIR>
__device__ __forceinline__ void load_weights(uint32_t dst, const CUtensorMap* m, uint32_t bar, const WeightBoxes& b,
                                             int step) {
  tma_load_4d_at<PAIR>(dst, m, bar, b.x + step * b.dx, b.y + step * b.dy, b.z, b.e);
  if (b.two) tma_load_4d_at<PAIR>(dst + kBK * 128, m, bar, b.x + 64, b.y + step * b.dy, b.z, b.e);
}

template <int CG, int TM, int STAGES, bool LORA>
__global__ void __maxnreg__(CG == 1 && LORA ? 96 : 168)
    gemm_grouped_sm100(const __grid_constant__ GroupedMaps maps, const __grid_constant__ GroupedParams p) {
  using Plan = GroupedPlan<CG, TM, STAGES, LORA>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sW = smem + Plan::kOffW;
  uint8_t* sT = smem + Plan::kOffT;
  uint8_t* sOut = smem + Plan::kOffOut;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Plan::kOffBar);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* land_bar = empty_bar + STAGES;   // an adapter's weights, per CTA
  uint64_t* built_bar = land_bar + STAGES;   // ... and its rows of h are in place, on the even CTA
  uint64_t* tfull_bar = built_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* rx_full = tempty_bar + 2;        // the cluster's sums for this CTA have arrived
  uint64_t* list_bar = rx_full + 1;          // the tile's adapters are listed
  uint64_t* list_read_bar = list_bar + 1;    // both producers and the MMA warp are done with the list
  uint64_t* done_bar = list_read_bar + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Plan::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* odd_flags = reinterpret_cast<volatile int*>(tmem_slot + 2);   // three tiles in turn
  int* scan = reinterpret_cast<int*>(smem + Plan::kOffScan);
  int* grp_rows = reinterpret_cast<int*>(smem + Plan::kOffRows);
  int* grp_tiles = reinterpret_cast<int*>(smem + Plan::kOffTiles);

  // With adapters there is one group: the rest of the tables holds the
  // adapter of each row of the tile, the distinct ones, and their counts.
  int* row_ids = grp_rows + 4;
  int* list = grp_tiles + 4;
  volatile int* list_counts = scan;   // adapters; scratch after that

  const int warp = static_cast<int>(threadIdx.x >> 5);
  const int lane = static_cast<int>(threadIdx.x & 31);
  // CG = 2: position in the CTA pair.  CG = 1: the last tiles' K blocks are
  // split over the CTAs of a cluster (GroupedWalk).
  const int csize = static_cast<int>(cluster_nctarank());
  const int crank = static_cast<int>(cluster_ctarank());
  const int rank = (CG == 2) ? crank : 0;
  const bool leader = (rank == 0);
  const int worker = static_cast<int>(blockIdx.x) / csize;
  const int workers = static_cast<int>(gridDim.x) / csize;

  if (threadIdx.x == 64) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 2);   // the two producers of the (even) CTA
      mbar_init(&empty_bar[s], 1);
      mbar_init(&land_bar[s], 1);
      mbar_init(&built_bar[s], kGrpEpiWarps / 2 * CG);   // one epilogue group of every CTA
    }
    mbar_init(&tfull_bar[0], 1);
    mbar_init(&tfull_bar[1], 1);
    mbar_init(&tempty_bar[0], kGrpEpiWarps * CG);
    mbar_init(&tempty_bar[1], kGrpEpiWarps * CG);
    mbar_init(rx_full, 1);
    mbar_init(list_bar, 1);
    mbar_init(list_read_bar, leader ? 3 : 2);
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    for (int i = 0; i < 3; ++i) odd_flags[i] = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    if (p.kb_total > 0) {   // K = 0: no maps
      for (int i = p.first_box; i < box_count(TM); ++i) prefetch_tmap(&maps.a[i]);
      prefetch_tmap(&maps.b);
    }
    if (LORA) prefetch_tmap(&maps.u);
    if (p.c_tma) prefetch_tmap(&maps.c);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc<CG>(tmem_slot, Plan::kTmemCols);
    tmem_relinquish<CG>();
  }
  tc_fence_before();
  __syncthreads();
  if (csize > 1) cluster_sync();   // the peers' barriers are initialised before any remote use
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // Parameters are read now, while the previous grid may still run: the
  // first read of each line of them costs a few hundred cycles.
  const int split_kb0 = p.kb_total * crank / csize, split_kb1 = p.kb_total * (crank + 1) / csize;
  asm volatile("" ::"l"(p.offsets), "r"(p.E), "r"(p.T), "r"(p.N), "r"(p.tiles_n), "r"(p.b_kmaj), "l"(p.bias), "l"(p.C),
               "r"(p.zero_rest), "r"(p.up_kmaj), "r"(split_kb0),
               "r"(split_kb1));
  // With LORA the previous grid is lora_shrink, whose CTAs let this one start
  // after their own wait, i.e. once everything before the call has completed:
  // the operands can be read at once, and only what touches h or C waits (the
  // epilogue warps, below).  (All waits at the start: 64 rows, 32 adapters of
  // rank 16, 4096 x 4096, 20.5 us against 17.9.)  A wait promises visibility to
  // the grid that waits.  This one relies on more: that what had completed
  // before its first CTA could start is in L2, where TMA reads and where the
  // indices and the bias are read from too (past L1).  Operands that this call
  // itself repacked, two launches before, are waited for.
  if (!LORA || p.packed) griddep_wait();
  const int rank_blocks = LORA ? (p.R + kLoraRanks - 1) / kLoraRanks : 0;

  auto tiles_of = [&](int n) { return (n + TM - 1) / TM * p.tiles_n; };
  if (p.offsets == nullptr || p.E > kWarpScanGroups ||
      !scan_groups_warp(p.offsets, p.off64, p.E, p.T, grp_rows, grp_tiles, tiles_of)) {
    scan_groups<kGrpThreads>(p.offsets, p.off64, p.E, p.T, grp_rows, grp_tiles, scan, p.err, tiles_of);
  }
  const int num_tiles = grp_tiles[p.E];
  GroupedWalk walk = grouped_walk<CG, Plan::kSubs>(num_tiles, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x),
                                                   worker, workers);
  int t;
  bool split = false;
  bool arrived = false;   // at the cluster barrier of the teardown

  if (warp == 0 || warp == kGrpRowsWarp) {
    // ------------------------------------------------------------ TMA producers: weights, rows
    if (lane == 0) {
      const bool weights = warp == 0;
      const uint32_t slot0 = smem_u32(weights ? sW : sT);
      const uint32_t slot_bytes = weights ? Plan::kWBytes : Plan::kTBytes;
      const uint32_t full0 = smem_u32(full_bar);
      const uint32_t even0 = CG == 2 ? mapa_shared(full0, 0) : full0;   // a pair's bytes complete on the even CTA
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      // per stage: parity of its last fill on full / land, and which came last
      uint32_t full_par = 0, land_par = 0, on_land = 0;
      bool ok = true;
      uint32_t list_phase = 0;
      // With LORA, what follows the first tile's K blocks waits for h in the end.
      // The bounded waits are for the work of this grid: the time that
      // lora_shrink takes is not theirs, so it is waited out first.
      bool first = true, waited = !LORA;
      auto wait_for_h = [&] {
        if (!waited) griddep_wait();
        waited = true;
      };
      while (ok && walk.next<Plan::kSubs>(t, split)) {
        if (!first) wait_for_h();
        first = false;
        const int parts = split ? csize : 1, part = split ? crank : 0;   // of the tile's K
        const int kb0 = split ? split_kb0 : 0, kb1 = split ? split_kb1 : p.kb_total;
        const GroupedUnit u = grouped_unit<CG, TM>(p, grp_rows, grp_tiles, t, walk.part);
        if (Plan::kSubs == 2 && u.rows == 0) continue;
        const int bcol = (u.tn * CG + rank) * kGrpCols;
        // the smallest box that holds this CTA's rows
        auto box_of = [&](int half) {
          int box = p.first_box;
          while (box + 1 < box_count(TM) && half <= box_rows(TM, box + 1)) ++box;
          return box;
        };
        const int half = u.nmma / CG, box = box_of(half);
        const int arow = u.row0 + rank * half;
        const CUtensorMap* map_a = &maps.a[box];
        uint32_t bytes = weights ? Plan::kWBytes : static_cast<uint32_t>(box_rows(TM, box)) * 128u;
        int arow2 = 0;
        const CUtensorMap* map_a2 = nullptr;
        if (Plan::kSubs == 2 && u.subs == 2) {
          GroupedUnit v = u;
          v.template second<Plan::kStep>();
          const int box2 = box_of(v.nmma / CG);
          arow2 = v.row0 + rank * (v.nmma / CG);
          map_a2 = &maps.a[box2];
          if (!weights) bytes += static_cast<uint32_t>(box_rows(TM, box2)) * 128u;
        }
        const WeightBoxes wb = weight_boxes(p.b_kmaj != 0, p.b_wide != 0, kb0 * kBK, bcol, u.e);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (issued >= STAGES && !mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], CG * bytes);
          const uint32_t dst = slot0 + stage * slot_bytes, bar = even0 + stage * 8;
          if (weights) {
            load_weights<CG == 2>(dst, &maps.b, bar, wb, kb - kb0);
          } else {
            tma_load_2d_at<CG == 2>(dst, map_a, bar, kb * kBK, arow);
            if (Plan::kSubs == 2 && map_a2) {
              tma_load_2d_at<CG == 2>(dst + Plan::kSubBytes, map_a2, bar, kb * kBK, arow2);
            }
          }
          full_par ^= 1u << stage;
          on_land &= ~(1u << stage);
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if constexpr (LORA) {
          ok = ok && mbar_wait(list_bar, list_phase, abort_flag);
          list_phase ^= 1u;
          const int adapters = ok ? list_counts[0] : 0;
          const int blocks = rank_blocks * adapters;
          const int b0 = blocks * part / parts, b1 = blocks * (part + 1) / parts;
          int rb = adapters ? b0 / adapters : 0, ai = b0 - rb * adapters;
          for (int b = b0; b < b1; ++b) {
            // the rows' producer loads nothing here, but has to see every phase
            // of a slot: two of them on, it would take an old one for its own
            if ((on_land >> stage) & 1u) wait_for_h();   // the slot's last block is multiplied with h
            if (issued >= STAGES && !mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag)) {
              ok = false;
              break;
            }
            if (weights) {
              const int a = list[ai], r0 = rb * kLoraRanks;
              if (++ai == adapters) {
                ai = 0;
                ++rb;
              }
              // on a barrier of this CTA: its epilogue warps look the weights over
              mbar_arrive_expect_tx(&land_bar[stage], Plan::kWBytes);
              load_weights<false>(slot0 + stage * slot_bytes, &maps.u, smem_u32(&land_bar[stage]),
                                  weight_boxes(p.up_kmaj != 0, p.up_wide != 0, r0, bcol, a), 0);
            }
            land_par ^= 1u << stage;
            on_land |= 1u << stage;
            ++issued;
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
          mbar_arrive(list_read_bar);
        }
      }
      if (weights) griddep_launch_dependents();
      if (!ok) {
        *abort_flag = 1;
        atomicOr(p.err, kDevErrTimeoutProducer);
      }
      // every fill must have landed before the CTA exits (the odd CTA's fills
      // of the even one's barriers are covered by the cluster barrier at
      // teardown)
      for (int s = 0; s < min(issued, STAGES); ++s) {
        const uint32_t bit = 1u << s;
        if ((on_land & bit) ? !weights : !leader) continue;
        uint64_t* bar = (on_land & bit) ? &land_bar[s] : &full_bar[s];
        const uint32_t par = (((on_land & bit) ? land_par : full_par) & bit) ? 0u : 1u;   // of the last fill
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(bar, par)) {
          if (globaltimer_ns() - t0 > kWaitLimitNs) {
            atomicOr(p.err, kDevErrTimeoutTeardown);
            break;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && leader) {
      // Descriptors of stage 0 (strides of the two major orders: see
      // gemm_sm100_kernel.cuh); an address counts in 16 bytes in their lowest
      // field.
      const uint64_t w_desc = smem_desc_sw128(smem_u32(sW), p.b_kmaj ? 16 : kBK * 128, 1024);
      const uint64_t t_desc = smem_desc_sw128(smem_u32(sT), 16, 1024);
      const uint32_t w_next = (p.b_kmaj ? kUmmaK * 2 : kUmmaK * 128) >> 4;   // 16 of K on
      int stage = 0;
      uint32_t full_par = 0;   // per stage: parity of its next fill
      int acc = 0;                      // the next accumulator
      uint32_t acc_used = 0, acc_par = 0;   // per accumulator: used before; parity of its next release
      uint32_t built_par = 0, list_phase = 0;
      bool ok = true, waited = !LORA;
      while (ok && walk.next<Plan::kSubs>(t, split)) {
        const int parts = split ? csize : 1, part = split ? crank : 0;   // of the tile's K
        const int kb0 = split ? split_kb0 : 0, kb1 = split ? split_kb1 : p.kb_total;
        if (p.kb_total == 0) break;   // the epilogue writes act(bias) by itself
        const GroupedUnit u = grouped_unit<CG, TM>(p, grp_rows, grp_tiles, t, walk.part);
        if (Plan::kSubs == 2 && u.rows == 0) continue;
        const uint32_t idesc = idesc_16bit(kGrpCols * CG, u.nmma, p.b_kmaj == 0, false, p.bf16 != 0);
        const uint32_t idesc2 = Plan::kSubs == 2 ? idesc_16bit(kGrpCols * CG, (u.rest + 31) / 32 * 32, p.b_kmaj == 0,
                                                              false, p.bf16 != 0)
                                                 : 0u;
        // takes accumulator `a` once its last tile has been read out
        auto take_acc = [&](int a) {
          const uint32_t bit = 1u << a;
          if ((acc_used & bit) && !mbar_wait(&tempty_bar[a], (acc_par & bit) ? 1u : 0u, abort_flag)) return false;
          if (acc_used & bit) acc_par ^= bit;
          acc_used |= bit;
          tc_fence_after();
          return true;
        };
        if (!take_acc(acc)) {
          ok = false;
          break;
        }
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * Plan::kSubRows);
        const uint32_t d_tmem2 = tmem_base + static_cast<uint32_t>((acc ^ 1) * Plan::kSubRows);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full_bar[stage], (full_par >> stage) & 1u, abort_flag)) {
            ok = false;
            break;
          }
          full_par ^= 1u << stage;
          tc_fence_after();
          const uint64_t wd = w_desc + static_cast<uint32_t>(stage * (Plan::kWBytes >> 4));
          const uint64_t td = t_desc + static_cast<uint32_t>(stage * (Plan::kTBytes >> 4));
#pragma unroll
          for (int j = 0; j < kBK / kUmmaK; ++j) {
            mma_f16_ss<CG>(d_tmem, wd + j * w_next, td + j * (kUmmaK * 2 >> 4), idesc, (kb > kb0 || j > 0) ? 1u : 0u);
          }
          if (Plan::kSubs == 2 && u.subs == 2) {
            if (kb == kb1 - 1) mma_commit<CG>(&tfull_bar[acc]);   // its rows can be read out beside the second part's MMAs
            if (kb == kb0 && !take_acc(acc ^ 1)) {
              ok = false;
              break;
            }
#pragma unroll
            for (int j = 0; j < kBK / kUmmaK; ++j) {
              mma_f16_ss<CG>(d_tmem2, wd + j * w_next, td + (Plan::kSubBytes >> 4) + j * (kUmmaK * 2 >> 4), idesc2,
                             (kb > kb0 || j > 0) ? 1u : 0u);
            }
          }
          mma_commit<CG>(&empty_bar[stage]);
          if (++stage == STAGES) stage = 0;
        }
        if constexpr (LORA) {
          ok = ok && mbar_wait(list_bar, list_phase, abort_flag);
          if (!waited) griddep_wait();   // see the producers
          waited = true;
          list_phase ^= 1u;
          const uint32_t idesc_up = idesc_16bit(kGrpCols * CG, u.nmma, p.up_kmaj == 0, false, true);   // bf16 parts
          const uint64_t up_desc = smem_desc_sw128(smem_u32(sW), p.up_kmaj ? 16 : kBK * 128, 1024);
          const uint32_t up_next = (p.up_kmaj ? kUmmaK * 2 : kUmmaK * 128) >> 4;
          const uint32_t up_rest = (p.up_kmaj ? kLoraRanks * 2 : kLoraRanks * 128) >> 4;   // see prepare_up
          const int adapters = ok ? list_counts[0] : 0;
          mbar_arrive(list_read_bar);
          const int blocks = rank_blocks * adapters;
          const int b0 = blocks * part / parts, b1 = blocks * (part + 1) / parts;
          int next = adapters ? adapters - b0 % adapters : 0;   // blocks up to the next 32 ranks
          int ranks = p.R - (adapters ? b0 / adapters * kLoraRanks : 0);
          for (int b = b0; b < b1; ++b) {
            // `up` has landed, h is in place
            if (!(CG == 2 ? mbar_wait_cluster(&built_bar[stage], (built_par >> stage) & 1u, abort_flag)
                          : mbar_wait(&built_bar[stage], (built_par >> stage) & 1u, abort_flag))) {
              ok = false;
              break;
            }
            built_par ^= 1u << stage;
            tc_fence_after();
            const uint64_t ud = up_desc + static_cast<uint32_t>(stage * (Plan::kWBytes >> 4));
            const uint64_t hd = t_desc + static_cast<uint32_t>(stage * (Plan::kTBytes >> 4));
            // hi, and lo 64 bytes on, with both parts of an fp16 `up`
            auto rank_step = [&](uint64_t up16, uint64_t h16) {
              mma_f16_ss<CG>(d_tmem, up16, h16, idesc_up, 1u);
              mma_f16_ss<CG>(d_tmem, up16, h16 + 4, idesc_up, 1u);
              if (!p.bf16) {
                mma_f16_ss<CG>(d_tmem, up16 + up_rest, h16, idesc_up, 1u);
                mma_f16_ss<CG>(d_tmem, up16 + up_rest, h16 + 4, idesc_up, 1u);
              }
            };
            rank_step(ud, hd);
            if (ranks > kUmmaK) rank_step(ud + up_next, hd + 2);
            mma_commit<CG>(&empty_bar[stage]);
            if (++stage == STAGES) stage = 0;
            if (--next == 0) {
              next = adapters;
              ranks -= kLoraRanks;
            }
          }
        }
        if (!ok) break;
        mma_commit<CG>(&tfull_bar[Plan::kSubs == 2 && u.subs == 2 ? acc ^ 1 : acc]);
        if (u.subs == 1) acc ^= 1;
      }
      if (!ok) {
        *abort_flag = 1;
        atomicOr(p.err, kDevErrTimeoutMma);
      }
      mma_commit<CG>(done_bar);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(done_bar, 0)) {
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
          atomicOr(p.err, kDevErrTimeoutTeardown);
          break;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int ew = warp & 3;                 // TMEM lane quarter of this warp
    const int col = ew * 32 + lane;          // column inside this CTA's 128
    const int et = static_cast<int>(threadIdx.x) - 64;
    const int eg = et >> 7;                  // epilogue group
    const int gt = et & 127;                 // thread of the group
    const uint32_t group_bar = 2u + static_cast<uint32_t>(eg);
    const bool bf16 = p.bf16 != 0;
    const uint32_t tempty_remote0 = (CG == 2) ? mapa_shared(smem_u32(&tempty_bar[0]), 0) : 0u;
    const uint32_t built_remote0 = (CG == 2) ? mapa_shared(smem_u32(&built_bar[0]), 0) : 0u;
    int stage = 0;
    uint32_t land_par = 0;
    bool waited = !LORA;
    uint32_t listed = 0;   // tiles whose adapters were listed
    if (p.zero_rest) zero_rows(p, grp_rows[0], grp_rows[p.E], et, 32 * kGrpEpiWarps);
    int acc = 0, turn = 0;
    uint32_t acc_par = 0;   // per accumulator: parity of its next fill
    bool ok = true;
    auto release_acc = [&] {
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && p.kb_total > 0) {
        if constexpr (CG == 1) {
          mbar_arrive(&tempty_bar[acc]);
        } else {
          mbar_arrive_cluster_relaxed(tempty_remote0 + static_cast<uint32_t>(acc * 8));
        }
      }
      acc_par ^= 1u << acc;
      acc ^= 1;
    };
    GroupedUnit u;
    int sub = 1;   // the part of the tile that comes next
    u.subs = 1;
    while (true) {
      if (Plan::kSubs == 1 || sub == u.subs) {
        if (!walk.next<Plan::kSubs>(t, split)) break;
        u = grouped_unit<CG, TM>(p, grp_rows, grp_tiles, t, walk.part);
        sub = 1;
        if (Plan::kSubs == 2 && u.rows == 0) continue;
      } else {
        u.template second<Plan::kStep>();
        ++sub;
      }
      const int parts = split ? csize : 1, part = split ? crank : 0;   // of the tile's K
      const int kb0 = split ? split_kb0 : 0, kb1 = split ? split_kb1 : p.kb_total;
      const int n0 = (u.tn * CG + rank) * kGrpCols;
      const int n = n0 + col;
      const float bias =
          (p.bias != nullptr && n < p.N) ? from_16bit(__ldcg(p.bias + static_cast<long long>(u.e) * p.N + n), bf16) : 0.0f;
      bool got = true;
      int adapters = 0, b0 = 0, b1 = 0;   // of the tile; this piece's adapter blocks
      if constexpr (LORA) {
        // The distinct adapters of the tile's rows, in order of their first
        // row, while the K blocks are multiplied.
        bool bad = false;
        const int id = et < u.rows ? adapter_of(p.adapter, p.adapter64, u.row0 + et, p.L, bad) : -1;
        if (bad) atomicOr(p.err, kDevErrBadAdapter);
        row_ids[et] = id;
        const unsigned same = __match_any_sync(0xffffffffu, id);   // rows of this warp with the same adapter
        bool first = id >= 0 && (same & ((1u << lane) - 1u)) == 0u;
        named_bar_sync(1, 32 * kGrpEpiWarps);
#pragma unroll 1
        for (int i = 0; i < (et & ~31) && first; i += 4) {   // earlier warps' rows, four at a time
          const int4 v = *reinterpret_cast<const int4*>(row_ids + i);
          first = v.x != id && v.y != id && v.z != id && v.w != id;
        }
        const unsigned vote = __ballot_sync(0xffffffffu, first);
        if (lane == 0) list_counts[2 + (et >> 5)] = __popc(vote);
        named_bar_sync(1, 32 * kGrpEpiWarps);
        int at = __popc(vote & ((1u << lane) - 1u)), all = 0;
        for (int w = 0; w < kGrpEpiWarps; ++w) {
          const int c = list_counts[2 + w];
          at += w < (et >> 5) ? c : 0;
          all += c;
        }
        if (listed > 0) mbar_wait(list_read_bar, (listed - 1) & 1u, abort_flag);   // the previous tile's
        ++listed;
        if (first) list[at] = id;
        if (et == 0) list_counts[0] = all;
        named_bar_sync(1, 32 * kGrpEpiWarps);
        if (et == 0) mbar_arrive(list_bar);
        adapters = all;
        if (!waited) griddep_wait();   // from here on h, the workspace and C
        waited = true;
        // adapter rows of this CTA's share of the tile: a group builds every
        // other block, its thread gt row gt, or half the ranks of row gt % 64
        // where there are no more rows
        constexpr int kRanks = CG == 1 ? kLoraRanks / 2 : kLoraRanks;
        constexpr int kChunks = kRanks / 8;
        b0 = rank_blocks * adapters * part / parts;
        b1 = rank_blocks * adapters * (part + 1) / parts;
        const int half = u.nmma / CG;
        const int row = CG == 1 ? gt & 63 : gt, sub = CG == 1 ? gt >> 6 : 0;
        const int tr = rank * half + row;   // row of the tile
        const int mine = (row < half && tr < u.rows) ? row_ids[tr] : -1;
        const float* hrow = p.h + static_cast<long long>(u.row0 + tr) * p.h_pitch;
        stage = (stage + kb1 - kb0) % STAGES;
        uint4 own[2 * kChunks];
        int have = -1;   // rank block held in `own`
        int rb = adapters ? b0 / adapters : 0, ai = b0 - rb * adapters;
        for (int b = b0; b < b1; ++b) {
          if (((b - b0) & 1) == eg) {
            if (rb != have) {
              const int r0 = rb * kLoraRanks + sub * kRanks;
              if (mine >= 0) split_ranks<kRanks>(hrow + r0, p.h_pitch - r0, own);
              have = rb;
            }
            const bool is = mine >= 0 && list[ai] == mine;
            // the producer waited for the slot to be free before it loaded `up`
            got = mbar_wait(&land_bar[stage], (land_par >> stage) & 1u, abort_flag);
            got = __all_sync(0xffffffffu, got) != 0;
            if (!got) break;
            const int steps = p.R - rb * kLoraRanks > kUmmaK ? 2 : 1;   // of 16 ranks
            if (prepare_up(sW + stage * Plan::kWBytes, gt, steps, p.up_kmaj != 0, bf16)) odd_flags[turn] = 1;
            if (row < half && sub < steps) {
              uint8_t* dst = sT + stage * Plan::kTBytes + row * 128;
#pragma unroll
              for (int i = 0; i < 2 * kChunks; ++i) {
                const int c = (i < kChunks ? 0 : kLoraRanks / 8 - kChunks) + sub * kChunks + i;   // hi, then lo
                *reinterpret_cast<uint4*>(dst + ((c ^ (row & 7)) << 4)) = is ? own[i] : make_uint4(0u, 0u, 0u, 0u);
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if constexpr (CG == 1) {
                mbar_arrive(&built_bar[stage]);
              } else {
                fence_release_smem_cluster();
                mbar_arrive_cluster_relaxed(built_remote0 + static_cast<uint32_t>(stage * 8));
              }
            }
          }
          if (++ai == adapters) {
            ai = 0;
            ++rb;
          }
          land_par ^= 1u << stage;
          if (++stage == STAGES) stage = 0;
        }
        // the next tile's flag; its last readers passed the barrier before this one
        if (et == 0) odd_flags[turn == 2 ? 0 : turn + 1] = 0;
      }
      // One lane per warp waits for the accumulator; all warps then take the
      // same decision, so none is left at a later barrier.
      if (got && p.kb_total > 0 && lane == 0) got = mbar_wait(&tfull_bar[acc], (acc_par >> acc) & 1u, abort_flag);
      got = __shfl_sync(0xffffffffu, got ? 1 : 0, 0) != 0;
      ok = named_bar_and(1, 32 * kGrpEpiWarps, got);
      if (!ok) break;
      tc_fence_after();
      const bool odd = LORA && odd_flags[turn] != 0;
      turn = turn == 2 ? 0 : turn + 1;
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(ew * 32) << 16) + static_cast<uint32_t>(acc * Plan::kSubRows);

      auto finish = [&](float v, float bias) {
        v += bias;
        if (p.act == 1) v = v < 0.0f ? 0.0f : v;   // a NaN stays one
        if (p.act == 2) v = gelu(v);
        return v;
      };

      if constexpr (CG == 2) {
        // chunks of 32 rows, alternating between the epilogue groups
#pragma unroll 1
        for (int r0 = eg * kGrpChunk; r0 < u.rows; r0 += 2 * kGrpChunk) {
          float f[32];
          if (p.kb_total > 0) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(tbase + r0, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = 0.0f;
          }
          if (LORA && odd && n < p.N) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (r0 + i < u.rows) f[i] += nonfinite_terms(p, list, adapters, b0, b1, u.row0 + r0 + i, n);
            }
          }
          // the store issued from this buffer a chunk ago has read it
          uint8_t* buf = sOut + eg * Plan::kOutBytes;
          if (p.c_tma && gt == 0) bulk_wait_group_read<0>();
          named_bar_sync(group_bar, 128);
          const uint32_t dst = smem_u32(buf) + col * 2;
          if (p.act == 2) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              f[i] += bias;
              f[i + 1] += bias;
              gelu2(f[i], f[i + 1]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = finish(f[i], bias);
          }
          if (bf16) {
#pragma unroll
            for (int i = 0; i < 32; ++i) st_shared_u16(dst + i * (kGrpCols * 2), to_16bit(f[i], true));
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) st_shared_u16(dst + i * (kGrpCols * 2), to_16bit(f[i], false));
          }
          // A TMA store clips its box at the tensor's edge in units larger than
          // an element (with an odd N it wrote past the end of the rows), so an
          // edge tile goes by TMA only when the rows end on a 16-byte boundary.
          const bool whole = p.c_tma && r0 + kGrpChunk <= u.rows &&
                             (n0 + kGrpCols <= p.N || (n0 < p.N && p.N % 8 == 0));
          if (whole) fence_proxy_async_smem();
          named_bar_sync(group_bar, 128);
          if (whole) {
            if (gt == 0) {
              tma_store_2d(&maps.c, buf, n0, u.row0 + r0);
              bulk_commit_group();
            }
          } else {
            store_rows(p, buf, u.row0 + r0, min(kGrpChunk, u.rows - r0), n0, gt, 128);
          }
        }
        release_acc();
      } else {
        // Few rows: steps of 8, in loops that are not unrolled.  A small call
        // runs this once, and what it costs then is fetching the instructions
        // (the 32-row form above took 5000 cycles for the sums of two rows).
        uint8_t* buf = sOut;   // all rows of the tile
        auto read8 = [&](int r0, float (&f)[8]) {
          uint32_t v[8];
          tmem_ld_32x32b_x8(tbase + r0, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = p.kb_total > 0 ? __uint_as_float(v[i]) : 0.0f;
          if (LORA && odd && n < p.N) {
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
              if (r0 + i >= u.rows) break;
              const float extra = nonfinite_terms(p, list, adapters, b0, b1, u.row0 + r0 + i, n);
#pragma unroll
              for (int q = 0; q < 8; ++q) f[q] += q == i ? extra : 0.0f;
            }
          }
        };
        if (parts == 1) {
#pragma unroll 1
          for (int r0 = eg * 8; r0 < u.rows; r0 += 16) {
            float f[8];
            read8(r0, f);
            const uint32_t dst = smem_u32(buf) + static_cast<uint32_t>(r0 * kGrpCols + col) * 2u;
#pragma unroll
            for (int i = 0; i < 8; ++i) st_shared_u16(dst + i * (kGrpCols * 2), to_16bit(finish(f[i], bias), bf16));
          }
          release_acc();
        } else {
          // Every row's partial sums go to the CTA that finishes it: the tile
          // as fp32 rows into the ring, which is idle now (a split tile is its
          // CTA's last), and from there one bulk copy to each other CTA
          // (stores of single words took 4000 cycles for 64 rows).
          const int per = (u.rows + parts - 1) / parts;   // rows per CTA, at most TM / parts
          const int mine0 = min(part * per, u.rows), mine = min(per, u.rows - mine0);   // rows that this CTA finishes
          const uint32_t rx = smem_u32(smem + Plan::kOffRx), rx_bar = smem_u32(rx_full);
          constexpr uint32_t kRow = kGrpCols * 4;
          float* own = reinterpret_cast<float*>(sW);
          float* biases = reinterpret_cast<float*>(sT);
          if (et == 0 && mine > 0) mbar_arrive_expect_tx(rx_full, static_cast<uint32_t>((parts - 1) * mine) * kRow);
          if (eg == 0) biases[col] = bias;
#pragma unroll 1
          for (int r0 = eg * 8; r0 < u.rows; r0 += 16) {
            float f[8];
            read8(r0, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) own[(r0 + i) * kGrpCols + col] = f[i];
          }
          fence_proxy_async_smem();
          named_bar_sync(1, 32 * kGrpEpiWarps);
          if (et < parts && et != part) {
            const int rows_to = min(per, u.rows - et * per);
            if (rows_to > 0) {
              bulk_copy_dsmem(mapa_shared(rx + static_cast<uint32_t>(part * per) * kRow, et),
                              smem_u32(sW) + static_cast<uint32_t>(et * per) * kRow,
                              static_cast<uint32_t>(rows_to) * kRow, mapa_shared(rx_bar, et));
            }
          }
          if (mine > 0) ok = __all_sync(0xffffffffu, mbar_wait(rx_full, 0, abort_flag)) != 0;
          if (!ok) break;
          cluster_arrive();   // what peers had for this CTA is here
          arrived = true;
          // 8 columns of a row per thread
          const float* sums = reinterpret_cast<const float*>(smem + Plan::kOffRx);
          const int seg = (et & 15) * 8;
          const int valid = min(8, p.N - n0 - seg);   // of them inside C
#pragma unroll 1
          for (int r = et >> 4; r < mine; r += 2 * kGrpEpiWarps) {
            float v[8] = {};
#pragma unroll 1
            for (int c = 0; c < parts; ++c) {   // in CTA order
              const float4* from = reinterpret_cast<const float4*>(
                  (c == part ? own + (mine0 + r) * kGrpCols : sums + (c * per + r) * kGrpCols) + seg);
              const float4 x = from[0], y = from[1];
              v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
              v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = finish(v[i], biases[seg + i]);
            const uint4 packed = make_uint4(pack_16bit(v[0], v[1], bf16), pack_16bit(v[2], v[3], bf16),
                                            pack_16bit(v[4], v[5], bf16), pack_16bit(v[6], v[7], bf16));
            unsigned short* out = p.C + static_cast<long long>(u.row0 + mine0 + r) * p.ldc + n0 + seg;
            if (p.c_vec && valid == 8) {
              *reinterpret_cast<uint4*>(out) = packed;
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const uint32_t w = i < 2 ? packed.x : i < 4 ? packed.y : i < 6 ? packed.z : packed.w;
                if (i < valid) out[i] = static_cast<unsigned short>(i & 1 ? w >> 16 : w);
              }
            }
          }
          break;   // a split tile is the CTA's last
        }
        // the next tile's staging comes after its accumulator barrier
        named_bar_sync(1, 32 * kGrpEpiWarps);
        store_rows(p, buf, u.row0, u.rows, n0, et, 32 * kGrpEpiWarps);
      }
    }
    if (!ok) {
      *abort_flag = 1;
      atomicOr(p.err, kDevErrTimeoutEpilogue);
    }
    if (CG == 2 && p.c_tma && gt == 0) bulk_wait_group_read<0>();
  }

  // ------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (csize > 1) {   // no CTA leaves while a peer may still reach its shared memory
    if (!arrived) cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<CG>(tmem_base, Plan::kTmemCols);
  }
}


// ------------------------------------------------------------------- weight gradient
//
//   D[e] = A_e^T G_e,   A_e, G_e = rows off[e] .. off[e + 1] of A [T, M] and G [T, N]
//
// A 256 x 256 tile of D[e] per CTA pair; the reduction runs over the group's
// rows, 64 per pipeline stage.  Both operands are read as they are stored:
// their rows are the MMA's K and their columns its M and N, i.e. both are
// MN-major (64-column atoms of 64 rows x 128 bytes).
//
// The rows of a group end anywhere, and the stage that holds the last ones
// also holds the next group's first ones (or inf / NaN behind the last row).
// Those must be zero in BOTH operands, since 0 * inf is not 0.  So the last
// stage of a cut group lands on a barrier of its own, a warp of its own zeroes the
// rows up to the next multiple of 16 in shared memory (a row of an atom is
// 128 contiguous bytes whatever the swizzle, at most 15 rows x 4 atoms), and
// the MMA reads only ceil(rows / 16) of the stage's four K steps.  The loads
// run ahead, so the fix-up is off the critical path.
//
// Groups without rows give a zero matrix, written without any MMA.
//
// What bounds it: with few rows to a group, writing D (4096 rows over 64
// experts 2048 x 1024: 59 us, and 43 with no rows at all, for 268 MB); with
// many, what bounds the pair tiles above.  Rings of 3, 4 and 5 stages took 244,
// 220 and 216 us for 8192 rows over 8 experts 4096 x 4096; the fifth stage's
// shared memory stages the output instead.
constexpr int kWgradThreads = kGrpThreads + 32;
constexpr int kWgradFixWarp = kGrpThreads / 32;   // warp 0 produces A, warp kGrpRowsWarp G
constexpr int kWgradTile = 256;

struct WgradParams {
  const void* offsets;
  int off64;
  int E;
  int T, M, N;
  int tiles_m, tiles_n;
  int bf16;
  unsigned short* D;       // [E, M, N], pitch ldd, stride_d from one matrix to the next
  long long ldd, stride_d;
  int d_tma;               // D is TMA-addressable
  int a_wide, g_wide;      // columns a multiple of 64: both atoms in one box
  int* err;
};

template <int STAGES>
struct WgradPlan {
  static constexpr int kOpBytes = kBK * 128 * 2;         // 64 rows x 128 columns of one operand: two atoms
  static constexpr int kStageBytes = 2 * kOpBytes;
  static constexpr int kOutBytes = kStoreRows * kStoreCols * 2;
  static constexpr int kOffA = 0;
  static constexpr int kOffG = STAGES * kOpBytes;
  static constexpr int kOffOut = 2 * STAGES * kOpBytes;
  static constexpr int kOffBar = kOffOut + 2 * kGrpEpiWarps * kOutBytes;
  static constexpr int kNumBars = 4 * STAGES + 4 + 1;    // full, empty, land, fix, tmem_full[2], tmem_empty[2], done
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kOffScan = kOffMisc + 16;
  static constexpr int kOffRows = kOffScan + 64;
  static constexpr int kOffBlocks = kOffRows + (kMaxGroups + 1) * 4;
  static constexpr int kUsed = kOffBlocks + (kMaxGroups + 1) * 4;
  static constexpr int kDynamicBytes = kUsed + 1024;
  static_assert(kDynamicBytes <= 227 * 1024, "shared memory of one CTA");
};

struct WgradUnit {
  int e, tm, tn;
  int row0, rows;   // the group's rows
  int blocks;       // ceil(rows / 64)
  int tail;         // rows of the last block when it is cut, else 0
};

__device__ __forceinline__ WgradUnit wgrad_unit(const WgradParams& p, const int* rows, int t) {
  WgradUnit u;
  const int tpe = p.tiles_m * p.tiles_n;
  u.e = t / tpe;
  const int local = t - u.e * tpe;
  const int per = kGrpRaster * p.tiles_n;
  const int g = local / per;
  const int gs = min(p.tiles_m - g * kGrpRaster, kGrpRaster);
  const int r = local - g * per;
  u.tm = g * kGrpRaster + r % gs;
  u.tn = r / gs;
  u.row0 = rows[u.e];
  u.rows = rows[u.e + 1] - u.row0;
  u.blocks = (u.rows + kBK - 1) / kBK;
  u.tail = u.rows % kBK;
  return u;
}

// 64 rows x 128 columns of an operand (see weight_boxes on the box count).
template <bool PAIR>
__device__ __forceinline__ void load_columns(uint32_t dst, const CUtensorMap* m, uint32_t bar, bool wide, int col,
                                             int row) {
  tma_load_3d_at<PAIR>(dst, m, bar, wide ? 0 : col, row, wide ? col >> 6 : 0);
  if (!wide) tma_load_3d_at<PAIR>(dst + kBK * 128, m, bar, col + 64, row, 0);
}

template <int STAGES>
__global__ void __launch_bounds__(kWgradThreads, 1)
    gemm_grouped_wgrad_sm100(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmG,
                             const __grid_constant__ CUtensorMap tmD, const __grid_constant__ WgradParams p) {
  using Plan = WgradPlan<STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem + Plan::kOffA;
  uint8_t* sG = smem + Plan::kOffG;
  uint8_t* sOut = smem + Plan::kOffOut;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Plan::kOffBar);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* land_bar = empty_bar + STAGES;   // a cut stage's bytes, per CTA
  uint64_t* fix_bar = land_bar + STAGES;     // ... zeroed, on the even CTA
  uint64_t* tfull_bar = fix_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint64_t* done_bar = tempty_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Plan::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* scan = reinterpret_cast<int*>(smem + Plan::kOffScan);
  int* grp_rows = reinterpret_cast<int*>(smem + Plan::kOffRows);
  int* grp_blocks = reinterpret_cast<int*>(smem + Plan::kOffBlocks);

  const int warp = static_cast<int>(threadIdx.x >> 5);
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int rank = static_cast<int>(cluster_ctarank());
  const bool leader = (rank == 0);
  const int worker = static_cast<int>(blockIdx.x) / 2;
  const int workers = static_cast<int>(gridDim.x) / 2;

  if (threadIdx.x == 64) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 2);   // the two producers of the even CTA
      mbar_init(&empty_bar[s], 1);
      mbar_init(&land_bar[s], 2);
      mbar_init(&fix_bar[s], 2);
    }
    mbar_init(&tfull_bar[0], 1);
    mbar_init(&tfull_bar[1], 1);
    mbar_init(&tempty_bar[0], kGrpEpiWarps * 2);
    mbar_init(&tempty_bar[1], kGrpEpiWarps * 2);
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmG);
    if (p.d_tma) prefetch_tmap(&tmD);
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc<2>(tmem_slot, 512);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  scan_groups<kWgradThreads>(p.offsets, p.off64, p.E, p.T, grp_rows, grp_blocks, scan, p.err,
                             [](int n) { return (n + kBK - 1) / kBK; });
  const int num_tiles = p.E * p.tiles_m * p.tiles_n;

  if (warp == 0 || warp == kGrpRowsWarp) {
    // ------------------------------------------------------------ TMA producers: A, G
    if (lane == 0) {
      const bool first = warp == 0;
      const CUtensorMap* map = first ? &tmA : &tmG;
      const bool wide = first ? p.a_wide != 0 : p.g_wide != 0;
      const uint32_t slot0 = smem_u32(first ? sA : sG);
      const uint32_t even0 = mapa_shared(smem_u32(full_bar), 0);
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      // per stage: parity of its last whole / cut fill, and which came last
      uint32_t full_par = 0, land_par = 0, was_cut = 0;
      bool ok = true;
      for (int t = worker; ok && t < num_tiles; t += workers) {
        const WgradUnit u = wgrad_unit(p, grp_rows, t);
        const int col = (first ? u.tm : u.tn) * kWgradTile + rank * 128;
        for (int b = 0; b < u.blocks; ++b) {
          if (issued >= STAGES && !mbar_wait(&empty_bar[stage], phase ^ 1u, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t dst = slot0 + stage * Plan::kOpBytes;
          const int row = u.row0 + b * kBK;
          const uint32_t bit = 1u << stage;
          if (b == u.blocks - 1 && u.tail) {
            mbar_arrive_expect_tx(&land_bar[stage], Plan::kOpBytes);
            load_columns<false>(dst, map, smem_u32(&land_bar[stage]), wide, col, row);
            was_cut |= bit;
            land_par ^= bit;
          } else {
            if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * Plan::kOpBytes);
            load_columns<true>(dst, map, even0 + stage * 8, wide, col, row);
            was_cut &= ~bit;
            full_par ^= bit;
          }
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (first) griddep_launch_dependents();
      if (!ok) {
        *abort_flag = 1;
        atomicOr(p.err, kDevErrTimeoutProducer);
      }
      // every fill must have landed before the CTA exits (whole fills of the
      // odd CTA complete on the even one's barriers and are covered by the
      // cluster barrier at teardown)
      for (int s = 0; s < min(issued, STAGES); ++s) {
        const uint32_t bit = 1u << s;
        if (!(was_cut & bit) && !leader) continue;
        uint64_t* bar = (was_cut & bit) ? &land_bar[s] : &full_bar[s];
        const uint32_t par = (((was_cut & bit) ? land_par : full_par) & bit) ? 0u : 1u;   // of the last fill
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(bar, par)) {
          if (globaltimer_ns() - t0 > kWaitLimitNs) {
            atomicOr(p.err, kDevErrTimeoutTeardown);
            break;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && leader) {
      const uint32_t idesc = idesc_16bit(256, kWgradTile, true, true, p.bf16 != 0);
      int stage = 0;
      uint32_t full_par = 0, fix_par = 0;   // per stage: parity of its next whole / cut fill
      int acc = 0;
      uint32_t acc_phase = 0;
      int count = 0;
      bool ok = true;
      for (int t = worker; ok && t < num_tiles; t += workers) {
        const WgradUnit u = wgrad_unit(p, grp_rows, t);
        if (u.blocks == 0) continue;
        if (count >= 2 && !mbar_wait(&tempty_bar[acc], acc_phase ^ 1u, abort_flag)) {
          ok = false;
          break;
        }
        ++count;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * kWgradTile);
        for (int b = 0; b < u.blocks; ++b) {
          const uint32_t bit = 1u << stage;
          const bool cut = b == u.blocks - 1 && u.tail;
          const bool got = cut ? mbar_wait_cluster(&fix_bar[stage], (fix_par & bit) ? 1u : 0u, abort_flag)
                               : mbar_wait(&full_bar[stage], (full_par & bit) ? 1u : 0u, abort_flag);
          if (!got) {
            ok = false;
            break;
          }
          if (cut) fix_par ^= bit;
          else full_par ^= bit;
          tc_fence_after();
          const int steps = cut ? (u.tail + kUmmaK - 1) / kUmmaK : kBK / kUmmaK;
          const uint32_t a0 = smem_u32(sA + stage * Plan::kOpBytes);
          const uint32_t g0 = smem_u32(sG + stage * Plan::kOpBytes);
          for (int j = 0; j < steps; ++j) {
            mma_f16_ss<2>(d_tmem, smem_desc_sw128(a0 + j * (kUmmaK * 128), kBK * 128, 1024),
                          smem_desc_sw128(g0 + j * (kUmmaK * 128), kBK * 128, 1024), idesc, (b > 0 || j > 0) ? 1u : 0u);
          }
          mma_commit<2>(&empty_bar[stage]);
          if (++stage == STAGES) stage = 0;
        }
        if (!ok) break;
        mma_commit<2>(&tfull_bar[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok) {
        *abort_flag = 1;
        atomicOr(p.err, kDevErrTimeoutMma);
      }
      mma_commit<2>(done_bar);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(done_bar, 0)) {
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
          atomicOr(p.err, kDevErrTimeoutTeardown);
          break;
        }
      }
    }
  } else if (warp == kWgradFixWarp) {
    // ------------------------------------------------------------ cut stages: zero the rows of others
    int stage = 0;
    uint32_t land_par = 0;
    for (int t = worker; t < num_tiles; t += workers) {
      const WgradUnit u = wgrad_unit(p, grp_rows, t);
      if (u.blocks == 0) continue;
      const int last = (stage + u.blocks - 1) % STAGES;
      stage = (last + 1) % STAGES;
      if (!u.tail) continue;
      const uint32_t bit = 1u << last;
      bool got = true;
      if (lane == 0) got = mbar_wait(&land_bar[last], (land_par & bit) ? 1u : 0u, abort_flag);
      got = __shfl_sync(0xffffffffu, got ? 1 : 0, 0) != 0;
      if (!got) {
        if (lane == 0) {
          *abort_flag = 1;
          atomicOr(p.err, kDevErrTimeoutProducer);
        }
        break;
      }
      land_par ^= bit;
      const int bytes = ((u.tail + kUmmaK - 1) / kUmmaK * kUmmaK - u.tail) * 128;   // per atom
      for (int o = lane * 16; o < bytes; o += 32 * 16) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int at = last * Plan::kOpBytes + j * (kBK * 128) + u.tail * 128 + o;
          *reinterpret_cast<uint4*>(sA + at) = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(sG + at) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        fence_release_smem_cluster();
        mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&fix_bar[last]), 0));
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int ew = warp & 3;
    const bool bf16 = p.bf16 != 0;
    const uint32_t tempty_remote0 = mapa_shared(smem_u32(&tempty_bar[0]), 0);
    const int half = (warp - 2) >> 2;      // column half of this warp: the two warps of a lane quarter share its rows
    uint8_t* bufs = sOut + (warp - 2) * 2 * Plan::kOutBytes;   // two staging boxes in turn
    int turn = 0;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = worker; t < num_tiles; t += workers) {
      const WgradUnit u = wgrad_unit(p, grp_rows, t);
      if (u.blocks > 0) {
        // every warp for itself: nothing below waits for another epilogue warp
        ok = __all_sync(0xffffffffu, mbar_wait(&tfull_bar[acc], acc_phase, abort_flag)) != 0;
        if (!ok) break;
        tc_fence_after();
      }
      const uint32_t tbase =
          tmem_base + (static_cast<uint32_t>(ew * 32) << 16) + static_cast<uint32_t>(acc * kWgradTile);
      const int m0 = u.tm * kWgradTile + rank * 128 + ew * 32;
      unsigned short* out = p.D + static_cast<long long>(u.e) * p.stride_d;
#pragma unroll 1
      for (int c0 = half * (kWgradTile / 2); c0 < (half + 1) * (kWgradTile / 2); c0 += kStoreCols) {
        const int n0 = u.tn * kWgradTile + c0;
        if (n0 >= p.N || m0 >= p.M) break;
        float f[64];
        if (u.blocks > 0) {
          uint32_t v[2][32];
          tmem_ld_32x32b_x32(tbase + c0, v[0]);
          tmem_ld_32x32b_x32(tbase + c0 + 32, v[1]);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 64; ++i) f[i] = __uint_as_float(v[i >> 5][i & 31]);
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) f[i] = 0.0f;
        }
        const bool whole = p.d_tma && (n0 + kStoreCols <= p.N || p.N % 8 == 0);
        uint8_t* buf = bufs + turn * Plan::kOutBytes;
        turn ^= 1;
        // the store issued from this box two chunks ago has read it
        if (p.d_tma) {
          if (lane == 0) bulk_wait_group_read<1>();
          __syncwarp();
        }
        auto stage_row = [&](bool b) {   // one conversion for two values
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            *reinterpret_cast<uint4*>(buf + lane * 128 + ((c ^ (lane & 7)) << 4)) =
                make_uint4(pack_16bit(f[8 * c], f[8 * c + 1], b), pack_16bit(f[8 * c + 2], f[8 * c + 3], b),
                           pack_16bit(f[8 * c + 4], f[8 * c + 5], b), pack_16bit(f[8 * c + 6], f[8 * c + 7], b));
          }
        };
        if (bf16) stage_row(true);
        else stage_row(false);
        if (whole) fence_proxy_async_smem();
        __syncwarp();
        if (p.d_tma && lane == 0) {
          if (whole) tma_store_3d(&tmD, buf, n0, m0, u.e);
          bulk_commit_group();   // empty when the box is stored below: the count above stays per box
        }
        if (!whole) {
          for (int r = 0; r < kStoreRows && m0 + r < p.M; ++r) {
            unsigned short* drow = out + static_cast<long long>(m0 + r) * p.ldd;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = h * 32 + lane;
              if (n0 + c < p.N) {
                drow[n0 + c] = *reinterpret_cast<const unsigned short*>(buf + r * 128 + (((c >> 3) ^ (r & 7)) << 4) +
                                                                        (c & 7) * 2);
              }
            }
          }
          __syncwarp();
        }
      }
      if (u.blocks > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(tempty_remote0 + static_cast<uint32_t>(acc * 8));
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
    if (!ok) {
      *abort_flag = 1;
      atomicOr(p.err, kDevErrTimeoutEpilogue);
    }
    if (p.d_tma && lane == 0) bulk_wait_group_read<0>();
  }

  // ------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem_base, 512);
  }
}

}  // namespace idb
