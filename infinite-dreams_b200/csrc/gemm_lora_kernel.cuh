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
// runs on its own.  tcgen05 would need 128 TMEM lanes for R = 8..64 ranks and
// one tile per adapter.
//
//  * a cluster of up to 8 CTAs x 8 warps shares the K range of a tile of TT
//    rows; warp w of CTA c takes the 32-element slices c * 8 + w, + 64, ...
//  * the rows of the tile are ordered by adapter (a stable rank count in
//    shared memory); chunks of up to 8 * NT8 rows of one adapter are the MMA
//    N, the ranks are the MMA M;
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
// The kernel also lists the distinct adapters of each row tile of the second
// kernel, which needs one pass over `up` per listed adapter.
#pragma once
#include "sm100_ptx.cuh"

namespace idb {

constexpr int kShrinkWarps = 8;
constexpr int kShrinkThreads = 32 * kShrinkWarps;
constexpr int kShrinkSlice = 32;        // K elements per warp step: two MMAs deep
constexpr int kShrinkMaxRows = 32;      // rows of a tile
constexpr int kAdapterListPitch = 260;  // count, up to 256 adapters of a 256-row tile, ..., rows without one

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
  int tile_rows;        // TT <= kShrinkMaxRows
  int x_vec, down_vec;  // rows 16-byte aligned / rank vectors aligned
  int* lists;           // [list_tiles, kAdapterListPitch]
  int list_tiles, list_rows;
  int* err;
};

// adapter[t], or -1 for none.  An index past the last adapter counts as none.
__device__ __forceinline__ int adapter_of(const void* adapter, int adapter64, long long t, int L, bool& bad) {
  const long long v =
      adapter64 ? static_cast<const long long*>(adapter)[t] : static_cast<const int*>(adapter)[t];
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
// read as zero.
__device__ __forceinline__ uint4 load8(const unsigned short* src, int valid, bool vec) {
  if (valid >= 8 && vec) return *reinterpret_cast<const uint4*>(src);
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = i < valid ? src[i] : 0u;
  return make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
}

// The `down` fragments of one slice: a[m][half] holds rank (m, half) of this
// lane's quad row for its 8 K elements.
template <int RT, bool KMAJ>
__device__ __forceinline__ void load_down(const ShrinkParams& p, const unsigned short* d, int r0, int k, int g,
                                          uint4 (&a)[RT][2]) {
  const int kv = p.K - k;   // valid elements from k on (may exceed 8, or be negative)
  if constexpr (KMAJ) {
#pragma unroll
    for (int m = 0; m < RT; ++m) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = r0 + m * 16 + half * 8 + g;
        a[m][half] = r < p.R ? load8(d + r * p.ld_down + k, kv, p.down_vec != 0) : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  } else {
    constexpr int V = 2 * RT;   // adjacent ranks of this lane: r0 + V g ..
    const int r = r0 + V * g;
    unsigned short e[8][V];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned short* src = d + (k + j) * p.ld_down + r;
      if (j < kv && p.down_vec && r + V <= p.R) {
        if constexpr (V == 2) {
          const ushort2 w = *reinterpret_cast<const ushort2*>(src);
          e[j][0] = w.x;
          e[j][1] = w.y;
        } else if constexpr (V == 4) {
          const ushort4 w = *reinterpret_cast<const ushort4*>(src);
          e[j][0] = w.x;
          e[j][1] = w.y;
          e[j][2] = w.z;
          e[j][3] = w.w;
        } else {
          const uint4 w = *reinterpret_cast<const uint4*>(src);
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < V; ++i) e[j][i] = static_cast<unsigned short>(ww[i / 2] >> (16 * (i & 1)));
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) e[j][i] = (j < kv && r + i < p.R) ? src[i] : static_cast<unsigned short>(0);
      }
    }
#pragma unroll
    for (int m = 0; m < RT; ++m) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = 2 * m + half;
        a[m][half] = make_uint4(e[0][i] | (static_cast<uint32_t>(e[1][i]) << 16),
                                e[2][i] | (static_cast<uint32_t>(e[3][i]) << 16),
                                e[4][i] | (static_cast<uint32_t>(e[5][i]) << 16),
                                e[6][i] | (static_cast<uint32_t>(e[7][i]) << 16));
      }
    }
  }
}

// Distinct adapters of rows [row0, row0 + n), n <= 256, in order of their
// first row: list[0] = count, list[1..].  Called by all threads.
__device__ __forceinline__ void list_adapters(const ShrinkParams& p, int row0, int n, int* list, int* ids,
                                              int* warp_counts) {
  const int tid = static_cast<int>(threadIdx.x);
  bool bad = false;
  const int a = tid < n ? adapter_of(p.adapter, p.adapter64, row0 + tid, p.L, bad) : -1;
  ids[tid] = a;
  if (bad) atomicOr(p.err, kDevErrBadAdapter);
  __syncthreads();
  bool first = a >= 0;
  for (int i = 0; i < tid && first; ++i) first = ids[i] != a;
  const unsigned vote = __ballot_sync(0xffffffffu, first);
  if ((tid & 31) == 0) warp_counts[tid >> 5] = __popc(vote);
  __syncthreads();
  int at = __popc(vote & ((1u << (tid & 31)) - 1u));
  for (int w = 0; w < (tid >> 5); ++w) at += warp_counts[w];
  if (first) list[1 + at] = a;
  if (tid == 0) {
    int total = 0;
    for (int w = 0; w < kShrinkWarps; ++w) total += warp_counts[w];
    list[0] = total;
  }
  const int without = __syncthreads_count(tid < n && a < 0);
  if (tid == 0) list[kAdapterListPitch - 1] = without;
}

// grid.x: tiles x cluster size (the cluster is along x); grid.y: blocks of 16 RT ranks.
template <int RT, int NT8, bool KMAJ, bool BF16>
__global__ void __launch_bounds__(kShrinkThreads) lora_shrink(const __grid_constant__ ShrinkParams p) {
  constexpr int RB = 16 * RT;
  extern __shared__ float red[];   // [kShrinkWarps][tile_rows][RB]
  __shared__ int ids[kShrinkThreads];
  __shared__ int order[kShrinkMaxRows];
  __shared__ int warp_counts[kShrinkWarps];
  __shared__ int active_s;
  const int tid = static_cast<int>(threadIdx.x);
  const int warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
  const int cs = static_cast<int>(cluster_nctarank());
  const int crank = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / cs;
  const int r0 = static_cast<int>(blockIdx.y) * RB;
  const int row0 = tile * p.tile_rows;
  const int rows = min(p.tile_rows, p.T - row0);

  griddep_wait();
  // Everything before this grid is complete now, so the second kernel may
  // start reading x and W; it waits for this grid before it reads h.
  griddep_launch_dependents();

  if (tile < p.list_tiles && crank == 0 && blockIdx.y == 0) {
    const int first = tile * p.list_rows;
    list_adapters(p, first, min(p.list_rows, p.T - first), p.lists + static_cast<long long>(tile) * kAdapterListPitch,
                  ids, warp_counts);
    __syncthreads();
  }
  // rows of the tile ordered by adapter, those without one left out
  if (tid < 32) {
    bool bad = false;
    const int a = tid < rows ? adapter_of(p.adapter, p.adapter64, row0 + tid, p.L, bad) : -1;
    ids[tid] = a;
    __syncwarp();
    int at = 0;
    for (int i = 0; i < rows; ++i) at += (ids[i] >= 0) && (ids[i] < a || (ids[i] == a && i < tid));
    if (a >= 0) order[at] = tid;
    const unsigned vote = __ballot_sync(0xffffffffu, a >= 0);
    if (tid == 0) active_s = __popc(vote);
  }
  __syncthreads();
  const int active = active_s;
  float* mine = red + static_cast<size_t>(warp) * p.tile_rows * RB;
  const int slices = (p.K + kShrinkSlice - 1) / kShrinkSlice;

  for (int c0 = 0; c0 < active;) {
    const int a = ids[order[c0]];
    int c1 = c0 + 1;
    while (c1 < active && c1 < c0 + 8 * NT8 && ids[order[c1]] == a) ++c1;
    const unsigned short* d = p.down + static_cast<long long>(a) * p.stride_down;
    const unsigned short* xr[NT8];
#pragma unroll
    for (int j = 0; j < NT8; ++j) {
      const int i = c0 + j * 8 + g;
      xr[j] = i < c1 ? p.x + static_cast<long long>(row0 + order[i]) * p.ldx : nullptr;
    }
    float acc[RT][NT8][4];
#pragma unroll
    for (int m = 0; m < RT; ++m) {
#pragma unroll
      for (int j = 0; j < NT8; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.0f;
      }
    }
#pragma unroll 2
    for (int s = crank * kShrinkWarps + warp; s < slices; s += cs * kShrinkWarps) {
      const int k = s * kShrinkSlice + q * 8;
      uint4 da[RT][2];
      load_down<RT, KMAJ>(p, d, r0, k, g, da);
      uint4 xb[NT8];
#pragma unroll
      for (int j = 0; j < NT8; ++j) {
        xb[j] = xr[j] != nullptr ? load8(xr[j] + k, p.K - k, p.x_vec != 0) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int j = 0; j < NT8; ++j) {
        if (j > 0 && c0 + j * 8 >= c1) break;
#pragma unroll
        for (int m = 0; m < RT; ++m) {
          mma_m16n8k16<BF16>(acc[m][j], da[m][0].x, da[m][1].x, da[m][0].y, da[m][1].y, xb[j].x, xb[j].y);
          mma_m16n8k16<BF16>(acc[m][j], da[m][0].z, da[m][1].z, da[m][0].w, da[m][1].w, xb[j].z, xb[j].w);
        }
      }
    }
    // accumulator (rank row g / g + 8, row of x 2q / 2q + 1) -> mine[sorted row][rank]
#pragma unroll
    for (int m = 0; m < RT; ++m) {
#pragma unroll
      for (int j = 0; j < NT8; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int half = i >> 1;
          const int at = c0 + j * 8 + 2 * q + (i & 1);
          const int r = KMAJ ? m * 16 + half * 8 + g : 2 * RT * g + 2 * m + half;
          if (at < c1) mine[at * RB + r] = acc[m][j][i];
        }
      }
    }
    c0 = c1;
  }
  __syncthreads();
  // over the warps, in place of the first warp's partial
  for (int e = tid; e < active * RB; e += kShrinkThreads) {
    float v = red[e];
#pragma unroll
    for (int w = 1; w < kShrinkWarps; ++w) v += red[static_cast<size_t>(w) * p.tile_rows * RB + e];
    red[e] = v;
  }
  // over the cluster: CTA c finishes every cs-th element
  cluster_sync();
  const uint32_t base = smem_u32(red);
  for (int e = tid * cs + crank; e < active * RB; e += kShrinkThreads * cs) {
    float v = 0.0f;
    for (int c = 0; c < cs; ++c) {
      float o;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(o) : "r"(mapa_shared(base + e * 4, c)));
      v += o;
    }
    const int t = order[e / RB];
    const float s = p.scale != nullptr ? p.scale[ids[t]] : 1.0f;
    p.h[static_cast<long long>(row0 + t) * p.h_pitch + r0 + e % RB] = v * s;
  }
  cluster_sync();   // no CTA leaves while a peer may still read its partials
}

}  // namespace idb
