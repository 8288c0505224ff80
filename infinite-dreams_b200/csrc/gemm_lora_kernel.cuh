// First half of the low-rank adapters beside a shared projection, for sm_100a:
//
//   h[t, :] = scale[a] * x[t, :] * down[a],   a = adapter[t]   (fp32, T x R)
//
// gemm_grouped_kernel.cuh adds h[t, :] * up[a] to the accumulators of x * W.
//
// The product is thin (R columns), so its cost is reading x once and each
// adapter's `down` once; the tensor work is 2 T K R FLOP.  What it needs is
// many loads in flight, spread over the machine even for one row, and rows of
// one tile that pick different weights.  Hence mma.sync fragments (16 ranks x
// 8 rows x 16 K) loaded straight from global memory, with no shared-memory
// staging and no barrier in the loop: every warp owns 32-wide K slices and
// runs on its own, the next slice's loads (of the next adapter too) in flight
// behind the current one's MMAs.  tcgen05 would need 128 TMEM lanes for R =
// 8..64 ranks and one tile per adapter.
//
//  * a cluster of up to 8 CTAs x 8 warps shares the K range of a tile of up to
//    8 rows; warp w of CTA c takes the 32-element slices c * 8 + w, + 64, ...
//  * the rows of a tile are ordered by adapter; the rows of one adapter are the
//    MMA N, the ranks are the MMA M;
//  * both operands need 8 adjacent K elements per lane.  The order of K inside
//    an MMA does not matter as long as both agree, so lane q of a quad takes
//    elements 8q .. 8q + 7 of the slice: one 16-byte load per row of x, and
//    per rank of a `down` stored R x K.  A `down` stored K x R is read 2 * RT
//    adjacent ranks per K row and re-paired in registers; the ranks are then
//    permuted among the MMA's rows, which the store undoes;
//  * partial sums: registers -> shared memory per warp -> summed over the
//    warps -> over the cluster through distributed shared memory, always in
//    the same order.  No workspace, no atomics.
//
// That form is for few rows, where every load is its own latency.  With many
// rows it reads `down` again for every 8 of them and has one step's loads in
// flight per warp, so there (lora_shrink_wide) a CTA takes 64 or 256 rows and
// brings x and `down` through a ring in shared memory by cp.async: 4096 rows, 4
// adapters of rank 64, 4096 x 4096 take 125 us with the product, which alone
// takes 107.
#pragma once
#include "sm100_ptx.cuh"

namespace idb {

constexpr int kShrinkWarps = 8;
constexpr int kShrinkThreads = 32 * kShrinkWarps;
constexpr int kShrinkSlice = 32;        // K elements per warp step: two MMAs deep
constexpr int kShrinkMaxRows = 8;       // rows of a tile

struct ShrinkParams {
  const unsigned short* x;
  long long ldx;
  const unsigned short* down;
  long long ld_down, stride_down;
  const void* adapter;  // int32 or int64 [T]; negative: none
  int adapter64;
  const float* scale;   // [L] or null (1)
  float* h;             // [T, h_pitch]
  int h_pitch;
  int T, K, L, R;
  int tile_rows;        // rows of a cluster
  int tiles;            // clusters that cover the rows
  int* err;
};

// 16-rank tiles of a block, and the pitch of h (whole blocks).
inline int shrink_rank_tiles(int64_t R) { return R <= 16 ? 1 : (R <= 32 ? 2 : 4); }
inline int64_t shrink_pitch(int64_t R) {
  const int64_t block = 16 * shrink_rank_tiles(R);
  return (R + block - 1) / block * block;
}

// Launches the kernel on rows of x that are 16-byte aligned (gemm_lora_shrink.cu).
int launch_shrink(const ShrinkParams& p, bool kmaj, bool bf16, int sms, cudaStream_t stream);

// adapter[t], or -1 for none.  An index past the last adapter counts as none.
// Read past L1: the product's grid does so before it waits for the one before it.
__device__ __forceinline__ int adapter_of(const void* adapter, int adapter64, long long t, int L, bool& bad) {
  const long long v =
      adapter64 ? __ldcg(static_cast<const long long*>(adapter) + t) : __ldcg(static_cast<const int*>(adapter) + t);
  bad |= v >= L;
  return (v < 0 || v >= L) ? -1 : static_cast<int>(v);
}

template <bool BF16>
__device__ __forceinline__ void mma_m16n8k16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// 8 adjacent elements src[0..7] as four words; positions at or past `valid`
// read as zero.  VEC: src is 16-byte aligned and `valid` is 8 or more, or 0
// or less.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const unsigned short* src, int valid) {
  if constexpr (VEC) {
    return valid > 0 ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
  } else {
    uint32_t h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = i < valid ? src[i] : 0u;
    return make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
  }
}

// The operands of one slice as they were loaded.  KMAJ (`down` stored R x K):
// d[2 m + half] holds rank (m, half) of this lane's quad row for its 8 K
// elements.  Else d holds, for each of the 8 K elements, the 2 RT adjacent
// ranks of this lane, packed.
template <int RT>
struct Slice {
  uint4 d[2 * RT];
  uint4 x;
};

template <int RT, bool KMAJ, bool VEC>
__device__ __forceinline__ void load_slice(const ShrinkParams& p, const unsigned short* d, int xrow, int r0, int k,
                                           int g, Slice<RT>& s) {
  const int kv = p.K - k;   // valid elements from k on (may exceed 8, or be negative)
  if constexpr (KMAJ) {
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) {
      const int r = r0 + i * 8 + g;
      s.d[i] = load8<VEC>(d + r * p.ld_down + k, r < p.R ? kv : 0);
    }
  } else {
    constexpr int V = 2 * RT;   // ranks r0 + V g ..
    const int r = r0 + V * g;
    uint32_t w[8 * RT];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned short* src = d + (k + j) * p.ld_down + r;
      if constexpr (VEC) {   // aligned to V elements, R a multiple of V
        const bool in = j < kv && r < p.R;
        if constexpr (RT == 1) {
          w[j] = in ? *reinterpret_cast<const uint32_t*>(src) : 0u;
        } else if constexpr (RT == 2) {
          const uint2 v = in ? *reinterpret_cast<const uint2*>(src) : make_uint2(0u, 0u);
          w[2 * j] = v.x;
          w[2 * j + 1] = v.y;
        } else {
          const uint4 v = in ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
          w[4 * j] = v.x;
          w[4 * j + 1] = v.y;
          w[4 * j + 2] = v.z;
          w[4 * j + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const uint32_t lo = (j < kv && r + 2 * i < p.R) ? src[2 * i] : 0u;
          const uint32_t hi = (j < kv && r + 2 * i + 1 < p.R) ? src[2 * i + 1] : 0u;
          w[j * RT + i] = lo | (hi << 16);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) s.d[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
  s.x = load8<VEC>(p.x + static_cast<long long>(max(xrow, 0)) * p.ldx + k, xrow >= 0 ? kv : 0);
}

// MMA A fragments (row g, row g + 8) of rank tile m: four K pairs each.
template <int RT, bool KMAJ>
__device__ __forceinline__ void rank_fragments(const Slice<RT>& s, int m, uint4& lo, uint4& hi) {
  if constexpr (KMAJ) {
    lo = s.d[2 * m];
    hi = s.d[2 * m + 1];
  } else {
    // word m of element j holds ranks (2m, 2m + 1) of the lane: pair elements
    auto word = [&](int j) {
      const int at = j * RT + m;
      const uint4 v = s.d[at / 4];
      return at % 4 == 0 ? v.x : (at % 4 == 1 ? v.y : (at % 4 == 2 ? v.z : v.w));
    };
    lo = make_uint4(__byte_perm(word(0), word(1), 0x5410), __byte_perm(word(2), word(3), 0x5410),
                    __byte_perm(word(4), word(5), 0x5410), __byte_perm(word(6), word(7), 0x5410));
    hi = make_uint4(__byte_perm(word(0), word(1), 0x7632), __byte_perm(word(2), word(3), 0x7632),
                    __byte_perm(word(4), word(5), 0x7632), __byte_perm(word(6), word(7), 0x7632));
  }
}

// grid.x: tiles x cluster size (the cluster is along x); grid.y: blocks of 16
// RT ranks.  Registers: 56 for 16 ranks stored R x K, so that two CTAs leave an SM
// room for one of the product's (64 rows, 32 adapters of rank 16, 4096 x 4096:
// 18.1 us, 20.2 with 59, which count as 64); stored K x R that costs more than it
// brings (2000 rows of 64 adapters, K = 4096: 144 us, 126 with 64).  Up to 96 for 32
// ranks (2000 rows, 64 adapters: 108 us, 140 with 80).
template <int RT, bool KMAJ, bool BF16, bool VEC>
__global__ void __maxnreg__(RT == 1 ? (KMAJ ? 56 : 64) : RT == 2 ? 96 : 128) lora_shrink(const __grid_constant__ ShrinkParams p) {
  constexpr int RB = 16 * RT;
  extern __shared__ float red[];   // [kShrinkWarps][tile_rows][RB]
  __shared__ float rx[kShrinkMaxRows * RB];   // this CTA's elements from the cluster: [CTA][element / cs]
  __shared__ uint64_t rx_full;
  __shared__ int gave_up;
  __shared__ int order[kShrinkMaxRows];
  __shared__ int order_id[kShrinkMaxRows];
  __shared__ int active_s;
  const int tid = static_cast<int>(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int cs = static_cast<int>(cluster_nctarank());
  const int crank = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / cs;
  const int r0 = static_cast<int>(blockIdx.y) * RB;
  const int slices = (p.K + kShrinkSlice - 1) / kShrinkSlice;

  if (tid == 0) {
    mbar_init(&rx_full, kShrinkWarps * cs);
    gave_up = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (cs > 1) cluster_sync();   // every CTA's barrier is there before any remote arrival
  griddep_wait();
  // Everything before this grid is complete now, so the second kernel may
  // start reading x and W; it waits for this grid before it reads h.
  griddep_launch_dependents();

  // rows of the tile ordered by adapter (stable), those without one left out
  const int row0 = tile * p.tile_rows;
  if (warp == 0) {
    const int rows = min(p.tile_rows, p.T - row0);
    bool bad = false;
    const int a = lane < rows ? adapter_of(p.adapter, p.adapter64, row0 + lane, p.L, bad) : -1;
    int at = 0;
#pragma unroll 8
    for (int i = 0; i < rows; ++i) {
      const int o = __shfl_sync(0xffffffffu, a, i);
      at += (o >= 0 && (o < a || (o == a && i < lane))) ? 1 : 0;
    }
    if (a >= 0) {
      order[at] = lane;
      order_id[at] = a;
    }
    const unsigned vote = __ballot_sync(0xffffffffu, a >= 0);
    if (lane == 0) active_s = __popc(vote);
  }
  __syncthreads();
  const int active = active_s;
  float* mine = red + static_cast<size_t>(warp) * p.tile_rows * RB;

  // This warp's steps: every chunk of rows, and in it this warp's slices.
  const int s_first = crank * kShrinkWarps + warp, s_step = cs * kShrinkWarps;
  int c0 = 0, c1 = 0;            // rows of the chunk being loaded, in sorted order
  const unsigned short* d = nullptr;
  int xrow = -1;
  auto open_chunk = [&](int at) {
    c0 = c1 = at;
    if (at >= active) return false;
    const int a = order_id[at];
    while (c1 < active && order_id[c1] == a) ++c1;
    d = p.down + static_cast<long long>(a) * p.stride_down;
    xrow = c0 + g < c1 ? row0 + order[c0 + g] : -1;
    return true;
  };
  float acc[RT][4];
  auto clear = [&] {
#pragma unroll
    for (int m = 0; m < RT; ++m) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][i] = 0.0f;
    }
  };
  // accumulator (rank row g / g + 8, row of x 2q / 2q + 1) -> mine[sorted row][rank]
  auto flush = [&](int f0, int f1) {
#pragma unroll
    for (int m = 0; m < RT; ++m) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int half = i >> 1;
        const int at = f0 + 2 * q + (i & 1);
        const int r = KMAJ ? m * 16 + half * 8 + g : 2 * RT * g + 2 * m + half;
        if (at < f1) mine[at * RB + r] = acc[m][i];
      }
    }
  };
  clear();
  if (s_first < slices) {
    Slice<RT> buf[2];
    bool have = open_chunk(0);
    int s = s_first;
    auto load = [&](Slice<RT>& to) {
      load_slice<RT, KMAJ, VEC>(p, d, xrow, r0, s * kShrinkSlice + q * 8, g, to);
    };
    // loads the step after `cur` into `next`, then multiplies `cur`
    auto step = [&](const Slice<RT>& cur, Slice<RT>& next) {
      const int f0 = c0, f1 = c1;
      s += s_step;
      const bool last = s >= slices;   // of this chunk
      if (last) {
        s = s_first;
        have = open_chunk(c1);
      }
      if (have) load(next);
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        uint4 lo, hi;
        rank_fragments<RT, KMAJ>(cur, m, lo, hi);
        mma_m16n8k16<BF16>(acc[m], lo.x, hi.x, lo.y, hi.y, cur.x.x, cur.x.y);
        mma_m16n8k16<BF16>(acc[m], lo.z, hi.z, lo.w, hi.w, cur.x.z, cur.x.w);
      }
      if (last) {
        flush(f0, f1);
        clear();
      }
    };
    if (have) load(buf[0]);
    while (have) {   // two buffers in turn: a copy would wait for the loads
      step(buf[0], buf[1]);
      if (have) step(buf[1], buf[0]);
    }
  } else {
    for (bool have = open_chunk(0); have; have = open_chunk(c1)) flush(c0, c1);   // no slice: zeros
  }
  __syncthreads();
  // over the warps, in place of the first warp's partial
  for (int e = tid; e < active * RB; e += kShrinkThreads) {
    float v = red[e];
#pragma unroll
    for (int w = 1; w < kShrinkWarps; ++w) v += red[static_cast<size_t>(w) * p.tile_rows * RB + e];
    red[e] = v;
  }
  if (cs == 1) {
    for (int e = tid; e < active * RB; e += kShrinkThreads) {   // the elements this thread summed
      const int at = e / RB;
      const float scale = p.scale != nullptr ? p.scale[order_id[at]] : 1.0f;
      p.h[static_cast<long long>(row0 + order[at]) * p.h_pitch + r0 + e % RB] = red[e] * scale;
    }
    return;
  }
  // Over the cluster: element e is finished by CTA e % cs; every CTA sends it
  // its partial (a sender may leave; only the receiver waits).
  const uint32_t rx0 = smem_u32(rx);
  const int share = (active * RB + cs - 1) / cs;
  for (int e = tid; e < active * RB; e += kShrinkThreads) {
    st_dsmem_f32(mapa_shared(rx0 + static_cast<uint32_t>(crank * share + e / cs) * 4u, e % cs), red[e]);
  }
  __syncwarp();
  if (lane < cs) mbar_arrive_cluster(mapa_shared(smem_u32(&rx_full), lane));
  if (!mbar_wait_cluster(&rx_full, 0, &gave_up)) {
    gave_up = 1;
    if (lane == 0) atomicOr(p.err, kDevErrTimeoutEpilogue);
    // stays until every peer has left or is here too: none may write into the
    // shared memory of a CTA that is gone
    cluster_arrive();
    cluster_wait();
    return;
  }
  for (int e = tid * cs + crank; e < active * RB; e += kShrinkThreads * cs) {
    float v = 0.0f;
    for (int c = 0; c < cs; ++c) v += rx[c * share + e / cs];   // in CTA order
    const int at = e / RB;
    const float scale = p.scale != nullptr ? p.scale[order_id[at]] : 1.0f;
    p.h[static_cast<long long>(row0 + order[at]) * p.h_pitch + r0 + e % RB] = v * scale;
  }
}

// ------------------------------------------------------------------- many rows
//
// A CTA owns ROWS rows (256, or 64 while that leaves SMs idle) and 64 ranks, the
// CTAs of a cluster share K in blocks of 64.  Each distinct adapter of the rows is
// one pass over this CTA's K blocks: x [ROWS x 64] and down[a] [64 x 64] arrive by
// cp.async in a ring (rows of 128 bytes with their 16-byte chunks
// swizzled by the row, so that ldmatrix reads them without conflicts).  With 256
// rows each of the 8 warps multiplies 32 of them by all ranks, with 64 rows 32 of
// them by 16 ranks, unless none of them picked the adapter.  The rows that did
// keep the result.  What it moves: x once per distinct adapter of a tile (once,
// for long prompts), `down` once per tile.  What bounds it is the latency of a
// step (barrier, ldmatrix, mma.sync, 1 to 2 us), so few rows are spread thin.
constexpr int kWideRanks = 64;
constexpr int kWideK = 64;
template <int ROWS>
struct WidePlan {
  static constexpr int kStages = 4;
  static constexpr int kXBytes = ROWS * 128;
  static constexpr int kStageBytes = kXBytes + kWideRanks * 128;
  static constexpr int kBytes = kStages * kStageBytes + ROWS * kWideRanks * 4;   // and the sums
  static constexpr int kRowWarps = ROWS / 32;               // warps side by side in the rows
  static constexpr int kRankTiles = 4 * kRowWarps / kShrinkWarps;   // 16-rank tiles of a warp
};

// 16 bytes of which `valid` bytes (0..16) come from src and the rest is zero.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool TRANS>
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (TRANS) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  } else {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
  }
}

// Byte offset of 16-byte chunk c of row r in a tile of 128-byte rows.
__device__ __forceinline__ uint32_t wide_at(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }

// grid as lora_shrink's, tile_rows = ROWS; x and `down` rows 16-byte aligned.
template <int ROWS, bool KMAJ, bool BF16>
__global__ void __launch_bounds__(kShrinkThreads) lora_shrink_wide(const __grid_constant__ ShrinkParams p) {
  using Plan = WidePlan<ROWS>;
  extern __shared__ __align__(128) uint8_t wide_smem[];
  __shared__ __align__(16) int ids[kShrinkThreads];
  __shared__ int list[ROWS];
  __shared__ int warp_counts[kShrinkWarps];
  const int tid = static_cast<int>(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int cs = static_cast<int>(cluster_nctarank());
  const int crank = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / cs;
  const int r0 = static_cast<int>(blockIdx.y) * kWideRanks;
  const int row0 = tile * ROWS;
  const int rw = warp % Plan::kRowWarps;                         // which 32 rows,
  const int mw = warp / Plan::kRowWarps * Plan::kRankTiles;      // and from which 16 ranks on

  griddep_wait();
  griddep_launch_dependents();   // see lora_shrink

  const int rows = min(ROWS, p.T - row0);
  // the distinct adapters of the rows, in order of their first row
  bool bad = false;
  const int id = tid < rows ? adapter_of(p.adapter, p.adapter64, row0 + tid, p.L, bad) : -1;
  ids[tid] = id;
  const unsigned same = __match_any_sync(0xffffffffu, id);
  bool first = id >= 0 && (same & ((1u << lane) - 1u)) == 0u;
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < (tid & ~31) && first; i += 4) {   // earlier warps' rows, four at a time
    const int4 v = *reinterpret_cast<const int4*>(ids + i);
    first = v.x != id && v.y != id && v.z != id && v.w != id;
  }
  const unsigned vote = __ballot_sync(0xffffffffu, first);
  if (lane == 0) warp_counts[warp] = __popc(vote);
  __syncthreads();
  int at = __popc(vote & ((1u << lane) - 1u)), adapters = 0;
  for (int w = 0; w < kShrinkWarps; ++w) {
    at += w < warp ? warp_counts[w] : 0;
    adapters += warp_counts[w];
  }
  if (first) list[at] = id;
  __syncthreads();
  const int my_id = ids[rw * 32 + lane];   // of the warp's rows
  const uint32_t ring = smem_u32(wide_smem);
  float* sums = reinterpret_cast<float*>(wide_smem + Plan::kStages * Plan::kStageBytes);   // [ROWS][64]

  const int blocks = (p.K + kWideK - 1) / kWideK;
  const int kb0 = blocks * crank / cs, per = blocks * (crank + 1) / cs - kb0;
  const int steps = adapters * per;
  // What a thread copies of a step: chunk c of the rows (tid / 8) + 32 i of x and
  // of `down`.  Everything that repeats is counted on, not divided out: the loop
  // below has a barrier per step and nothing to hide a chain of divisions behind.
  const int c = tid & 7, r8 = tid >> 3;
  const uint32_t at0 = wide_at(r8, c);
  const unsigned short* xr = p.x + static_cast<long long>(row0 + r8) * p.ldx + c * 8;
  int l_block = 0, l_adapter = 0, l_stage = 0;
  auto load = [&] {   // x and down[a] of the next step into the next stage
    const int k0 = (kb0 + l_block) * kWideK;
    const uint32_t sx = ring + static_cast<uint32_t>(l_stage * Plan::kStageBytes), sd = sx + Plan::kXBytes;
    const int xv = max(0, min(8, p.K - k0 - c * 8)) * 2;   // valid bytes of this thread's chunks of x
#pragma unroll
    for (int i = 0; i < ROWS / 32; ++i) {
      const bool in = i * 32 + r8 < rows && xv > 0;
      cp_async_16(sx + at0 + i * 4096, in ? xr + static_cast<long long>(i * 32) * p.ldx + k0 : p.x, in ? xv : 0);
    }
    const unsigned short* d = p.down + static_cast<long long>(list[l_adapter]) * p.stride_down;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = i * 32 + r8;   // KMAJ: a rank, its K chunks; else a K row, its rank chunks
      int valid;
      const unsigned short* src;
      if constexpr (KMAJ) {
        valid = r0 + r < p.R ? xv : 0;
        src = d + static_cast<long long>(r0 + r) * p.ld_down + k0 + c * 8;
      } else {
        valid = k0 + r < p.K ? max(0, min(8, p.R - r0 - c * 8)) * 2 : 0;
        src = d + static_cast<long long>(k0 + r) * p.ld_down + r0 + c * 8;
      }
      cp_async_16(sd + at0 + i * 4096, valid > 0 ? src : p.x, valid);
    }
    if (++l_block == per) {
      l_block = 0;
      ++l_adapter;
    }
    if (++l_stage == Plan::kStages) l_stage = 0;
  };
  for (int s = 0; s < Plan::kStages - 1; ++s) {
    if (s < steps) load();
    cp_async_commit();
  }
  float acc[Plan::kRankTiles][4][4];   // [16 ranks][8 rows]
  const int rank_tiles = (p.R - r0 + 15) / 16 - mw;   // that exist, from the warp's first on; the others stay zero
  bool mine = false;    // a row of this warp picked the adapter
  int block = 0, adapter = 0, stage = 0;
  for (int step = 0; step < steps; ++step) {
    cp_async_wait<Plan::kStages - 2>();
    __syncthreads();   // every thread's part of this stage is in, and the stage about to be refilled is read
    if (step + Plan::kStages - 1 < steps) load();
    cp_async_commit();
    if (block == 0) {
      mine = __any_sync(0xffffffffu, my_id == list[adapter]);
#pragma unroll
      for (int m = 0; m < Plan::kRankTiles; ++m) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.0f;
        }
      }
    }
    if (mine) {
      const uint32_t sx = ring + static_cast<uint32_t>(stage * Plan::kStageBytes), sd = sx + Plan::kXBytes;
#pragma unroll
      for (int kk = 0; kk < kWideK / 16; ++kk) {
        // B: 8 rows x 16 K per pair of 8x8 blocks; blocks (rows j, K lo), (j, K hi), (j + 1, K lo), (j + 1, K hi)
        uint32_t xb[2][4];
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const int r = rw * 32 + jj * 16 + (lane & 7) + ((lane >> 4) << 3);
          ldmatrix_x4<false>(sx + wide_at(r, kk * 2 + ((lane >> 3) & 1)), xb[jj]);
        }
#pragma unroll
        for (int m = 0; m < Plan::kRankTiles; ++m) {
          if (m >= rank_tiles) break;
          // A: blocks (ranks 0-7, K lo), (8-15, K lo), (0-7, K hi), (8-15, K hi)
          uint32_t da[4];
          if constexpr (KMAJ) {
            const int r = (mw + m) * 16 + (lane & 15);
            ldmatrix_x4<false>(sd + wide_at(r, kk * 2 + (lane >> 4)), da);
          } else {
            const int k = kk * 16 + (lane & 7) + ((lane >> 4) << 3);
            ldmatrix_x4<true>(sd + wide_at(k, (mw + m) * 2 + ((lane >> 3) & 1)), da);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            mma_m16n8k16<BF16>(acc[m][j], da[0], da[1], da[2], da[3], xb[j >> 1][(j & 1) * 2], xb[j >> 1][(j & 1) * 2 + 1]);
          }
        }
      }
      if (block == per - 1) {
        const int a = list[adapter];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = rw * 32 + j * 8 + 2 * q + i;
            if (ids[r] == a) {
#pragma unroll
              for (int m = 0; m < Plan::kRankTiles; ++m) {
                sums[r * kWideRanks + (mw + m) * 16 + g] = acc[m][j][i];
                sums[r * kWideRanks + (mw + m) * 16 + 8 + g] = acc[m][j][i + 2];
              }
            }
          }
        }
      }
    }
    if (++block == per) {
      block = 0;
      ++adapter;
    }
    if (++stage == Plan::kStages) stage = 0;
  }
  // over the cluster, in CTA order: CTA c finishes every cs-th row, a thread four
  // ranks of it
  if (cs > 1) cluster_sync();
  else __syncthreads();
  const uint32_t base = smem_u32(sums);
  const int e = (tid & 15) * 4;
  if (r0 + e < p.h_pitch) {   // the pitch is whole blocks of 16
    auto store = [&](int r, float4 v) {
      const int a = ids[r];
      if (a < 0) return;
      const float scale = p.scale != nullptr ? p.scale[a] : 1.0f;
      *reinterpret_cast<float4*>(p.h + static_cast<long long>(row0 + r) * p.h_pitch + r0 + e) =
          make_float4(v.x * scale, v.y * scale, v.z * scale, v.w * scale);
    };
    if (cs == 1) {
#pragma unroll 4
      for (int r = tid >> 4; r < rows; r += kShrinkThreads / 16) {
        store(r, *reinterpret_cast<const float4*>(sums + r * kWideRanks + e));
      }
    } else {
#pragma unroll 1
      for (int r = (tid >> 4) * cs + crank; r < rows; r += kShrinkThreads / 16 * cs) {
        float4 part[8];   // in flight together
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (c < cs) part[c] = ld_dsmem_f32x4(mapa_shared(base + (r * kWideRanks + e) * 4, c));
        }
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          if (c < cs) v = make_float4(v.x + part[c].x, v.y + part[c].y, v.z + part[c].z, v.w + part[c].w);
        }
        store(r, v);
      }
    }
  }
  if (cs > 1) cluster_sync();   // no CTA leaves while a peer may still read its sums
}

}  // namespace idb
