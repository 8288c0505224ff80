// Launcher of lora_shrink (gemm_lora_kernel.cuh): picks the compiled variant
// and the grid.
#include <atomic>

#include "../../include/gemm_sm100.h"
#include "gemm_capi_shared.h"
#include "gemm_lora_kernel.cuh"

namespace idb {
namespace {

using ShrinkFn = void (*)(ShrinkParams);

// More rows than kWideFrom take lora_shrink_wide, if there are few adapters.  It
// passes over x once per distinct adapter of a tile, 64 ranks at a time, which only
// the device knows the number of; the number of adapters bounds it.  So up to 4
// adapters per 16 ranks of the other form's block.  Both forms, wide first, K =
// 4096 with a product of 128 columns, rows in long runs and every row another
// adapter, us:
//   8192 rows, rank 64:   16 adapters   54, 359     116, 518
//                         64            72, 1249    119, 625
//   8192 rows, rank 16:    4 adapters   46,  87      55, 120
//                         16            46, 249      55, 195
//                         64            58, 842      56, 226
//   32768 rows, rank 64:  16 adapters  167, 1370    406, 1860
//                        256           234, 12479   411, 2480
constexpr int kWideFrom = 2048;
constexpr int kWideAdapters = 4;

template <int RT, bool VEC>
ShrinkFn pick(bool kmaj, bool bf16) {
  if (kmaj) return bf16 ? lora_shrink<RT, true, true, VEC> : lora_shrink<RT, true, false, VEC>;
  return bf16 ? lora_shrink<RT, false, true, VEC> : lora_shrink<RT, false, false, VEC>;
}

template <int ROWS>
ShrinkFn pick_wide(bool kmaj, bool bf16) {
  if (kmaj) return bf16 ? lora_shrink_wide<ROWS, true, true> : lora_shrink_wide<ROWS, true, false>;
  return bf16 ? lora_shrink_wide<ROWS, false, true> : lora_shrink_wide<ROWS, false, false>;
}

}  // namespace

int launch_shrink(const ShrinkParams& sp, bool kmaj, bool bf16, int sms, cudaStream_t stream) {
  ShrinkParams p = sp;
  const int rt = shrink_rank_tiles(p.R);
  const int elems = kmaj ? 8 : 2 * rt;   // of `down` per load
  const bool vec = p.K % 8 == 0 && reinterpret_cast<uintptr_t>(p.down) % (2 * elems) == 0 && p.ld_down % elems == 0 &&
                   p.stride_down % elems == 0 && (kmaj || p.R % elems == 0);
  const bool aligned = reinterpret_cast<uintptr_t>(p.down) % 16 == 0 && p.ld_down % 8 == 0 && p.stride_down % 8 == 0;
  ShrinkFn fn;
  int cluster = 1, bytes, ranks, variant;
  if (p.T > kWideFrom && p.L <= kWideAdapters * rt && aligned) {
    // 256 rows to a cluster if that gives at least half of the SMs a CTA, else
    // 64; as many CTAs along K as keep to one (two) per SM with at least 4 K
    // blocks each.  With the product, rank 64: 8192 rows in long runs, 4096 x
    // 4096, 245 us against 254 with 64 rows; 4096 rows, 1024 x 1024, 33 against
    // 44 with 256.
    ranks = kWideRanks;
    const int blocks = (p.K + kWideK - 1) / kWideK, rank_blocks = (p.R + ranks - 1) / ranks;
    auto tiles_of = [&](int rows) { return (p.T + rows - 1) / rows; };
    auto cluster_of = [&](int64_t ctas, int most) {
      int c = 1;
      while (c < 8 && 8 * c <= blocks && 2 * c * ctas <= most) c *= 2;
      return c;
    };
    const int64_t tall_ctas = static_cast<int64_t>(tiles_of(256)) * rank_blocks;
    const bool tall = 2 * tall_ctas * cluster_of(tall_ctas, sms) >= sms;
    p.tile_rows = tall ? 256 : 64;
    p.tiles = tiles_of(p.tile_rows);
    cluster = cluster_of(static_cast<int64_t>(p.tiles) * rank_blocks, tall ? sms : 2 * sms);
    fn = tall ? pick_wide<256>(kmaj, bf16) : pick_wide<64>(kmaj, bf16);
    bytes = tall ? WidePlan<256>::kBytes : WidePlan<64>::kBytes;
    variant = tall * 4 + kmaj * 2 + bf16;
  } else {
    // So few rows to a tile that two CTAs per SM share the work (T = 64: 2 rows
    // x 32 clusters of 8), up to the 8 rows of one MMA; along K no more CTAs
    // than give every warp a slice.
    int rows = 1;
    while (rows < 8 && rows * 32 < p.T) rows *= 2;
    p.tile_rows = rows;
    p.tiles = (p.T + rows - 1) / rows;
    ranks = 16 * rt;
    const int slices = (p.K + kShrinkSlice - 1) / kShrinkSlice;
    while (cluster < 8 && cluster * kShrinkWarps < slices && cluster * p.tiles <= sms) cluster *= 2;
    // operands without vector alignment take the element-wise loads
    fn = rt == 1   ? (vec ? pick<1, true>(kmaj, bf16) : pick<1, false>(kmaj, bf16))
         : rt == 2 ? (vec ? pick<2, true>(kmaj, bf16) : pick<2, false>(kmaj, bf16))
                   : (vec ? pick<4, true>(kmaj, bf16) : pick<4, false>(kmaj, bf16));
    variant = 8 + (rt == 4 ? 2 : rt - 1) * 8 + vec * 4 + kmaj * 2 + bf16;
    bytes = kShrinkWarps * rows * ranks * static_cast<int>(sizeof(float));   // at most 16 KiB
  }
  // Once per kernel and device: the dynamic shared memory above 48 KiB, and the
  // SM's largest shared-memory split.  The product's CTA needs that split, and
  // an SM changes it only when it is empty: under a smaller one the product's
  // CTAs did not start before this grid had ended.
  static std::atomic<unsigned long long> configured[32];   // devices, per variant
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return capi_fail_cuda(e, "cudaGetDevice");
  const unsigned long long bit = 1ull << (dev & 63);
  if (!(configured[variant].load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess && bytes > 48 * 1024) {
      e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    }
    if (e != cudaSuccess) return capi_fail_cuda(e, "adapter kernel attribute");
    configured[variant].fetch_or(bit, std::memory_order_acq_rel);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.tiles * cluster),
                     static_cast<unsigned>((p.R + ranks - 1) / ranks), 1);
  cfg.blockDim = dim3(kShrinkThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, fn, p);
  return e == cudaSuccess ? GEMM_OK : capi_fail_cuda(e, "adapter kernel launch");
}

}  // namespace idb
