// C ABI of the products whose weight is picked by the row (declared in
// include/gemm_sm100.h): validation, repacking of operands that TMA cannot
// address, tensor maps and launches, in the manner of gemm_capi.cu.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <string>

#include "../../include/gemm_sm100.h"
#include "gemm_capi_shared.h"
#include "gemm_grouped_kernel.cuh"
#include "gemm_pack.cuh"

namespace idb {

// The operands of a call that TMA cannot address, repacked in one launch: a
// dependent of the grid before it and the grid after it its dependent, so the
// launches overlap.  1000 rows by 5 x 777 x 1023 weights: 20 us with the
// repacking, 12 us for 5 x 776 x 1024, which needs none.
//
// A CTA takes slabs of 256 PER chunks of one matrix, all of a thread's loads in
// flight together; PER = 4 where that leaves every SM two CTAs, else 1 (1879
// rows by 94 x 4224 x 278 stored N x K: 172 us against 210 with one chunk and
// its index divisions at a time; 64 rows by 777 x 1024: 11 us).  Matrices whose group is empty are left out: no tile reads
// them.  (Offsets out of order are clamped upwards by the product, which only
// empties more groups.)
constexpr int kPackThreads = 256;

template <int PER, class Index>
__device__ __forceinline__ void pack_slab(const PackJob& job, int b, Index first) {
  const Index chunks = static_cast<Index>((job.cols + 7) / 8), total = chunks * static_cast<Index>(job.rows);
  const uintptr_t begin = reinterpret_cast<uintptr_t>(job.src) + static_cast<uintptr_t>(b * job.stride) * 2u;
  const uintptr_t end = begin + (static_cast<uintptr_t>(job.rows - 1) * static_cast<uintptr_t>(job.lds) + job.cols) * 2u;
  unsigned short* dst = static_cast<unsigned short*>(job.dst) + static_cast<long long>(b) * job.rows * job.ldd;
  uint4 v[PER];
  long long to[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const Index i = first + k * kPackThreads + threadIdx.x;
    to[k] = -1;
    if (i < total) {
      const Index r = i / chunks;
      const int c = static_cast<int>(i - r * chunks) * 8;
      to[k] = static_cast<long long>(r) * job.ldd + c;
      v[k] = pack_chunk(begin, end, begin + static_cast<uintptr_t>(static_cast<long long>(r) * job.lds + c) * 2u, job.cols - c);
    }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    if (to[k] >= 0) *reinterpret_cast<uint4*>(dst + to[k]) = v[k];
  }
}

// Slabs of one matrix of the job.
__host__ __device__ inline long long pack_slabs(const PackJob& job, int slab) {
  return (static_cast<long long>(job.rows) * ((job.cols + 7) / 8) + slab - 1) / slab;
}

template <int PER>
__global__ void __launch_bounds__(kPackThreads) pack_stacks(const __grid_constant__ PackJobs jobs) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kSlab = kPackThreads * PER;
  for (int j = 0; j < jobs.count; ++j) {
    const PackJob& job = jobs.job[j];
    const long long slabs = pack_slabs(job, kSlab);
    for (long long s = blockIdx.x; s < slabs * job.batch; s += gridDim.x) {
      const int b = static_cast<int>(s / slabs);
      if (job.offsets != nullptr) {
        const bool rows = job.off64 ? static_cast<const long long*>(job.offsets)[b + 1] > static_cast<const long long*>(job.offsets)[b]
                                    : static_cast<const int*>(job.offsets)[b + 1] > static_cast<const int*>(job.offsets)[b];
        if (!rows) continue;
      }
      const long long first = (s - b * slabs) * kSlab;
      if (slabs * kSlab < (1ll << 31)) pack_slab<PER, uint32_t>(job, b, static_cast<uint32_t>(first));
      else pack_slab<PER, unsigned long long>(job, b, static_cast<unsigned long long>(first));
    }
  }
}

namespace {

constexpr int64_t kInt32Max = (1ll << 31) - 1;

// Largest extent of a call: the kernels round rows and columns up to whole tiles
// (at most 512) and step by the grid, in 32 bits.
constexpr int64_t kMaxExtent = (1ll << 31) - 1024;

int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// One operand: `batch` matrices of rows x cols, pitch ld, `stride` elements
// from one matrix to the next.
struct Operand {
  const void* p = nullptr;
  int64_t batch = 1, rows = 0, cols = 0, ld = 0, stride = 0;
  size_t pack_off = 0;
  bool pack = false;

  Operand(const void* ptr, int64_t b, int64_t r, int64_t c, int64_t l, int64_t s)
      : p(ptr), batch(b), rows(r), cols(c), ld(l), stride(s) {}

  // Reserves workspace for a copy when TMA cannot address the operand as it
  // is (16-byte base, row pitch and matrix stride).  The copy's rows are
  // padded to 64 elements, one 128-byte line per TMA box row, as in gemm_launch.
  void plan(size_t* off) {
    const bool ok = reinterpret_cast<uintptr_t>(p) % 16u == 0 && ld % 8 == 0 &&
                    (batch == 1 || (stride % 8 == 0 && stride > 0));
    pack = !ok && batch > 0 && rows > 0 && cols > 0;
    if (!pack) return;
    pack_off = *off;
    *off = align256(*off + static_cast<size_t>(batch) * rows * round_up(cols, 64) * 2);
  }

  // Adds the copy to `jobs` and describes it from now on; with offsets, the
  // matrices of empty groups are left out.
  void add(uint8_t* ws, PackJobs* jobs, const void* offsets = nullptr, int off64 = 0) {
    if (!pack) return;
    const int64_t ldp = round_up(cols, 64);
    jobs->job[jobs->count++] = {p, ld, batch == 1 ? 0 : stride, ws + pack_off, ldp, static_cast<int>(batch),
                                static_cast<int>(rows), static_cast<int>(cols), offsets, off64};
    p = ws + pack_off;
    ld = ldp;
    stride = rows * ldp;
  }

  // Boxes of `box_rows` rows x 64 columns.
  int encode_rows(CUtensorMap* m, int box_rows, const char* what) const {
    const int64_t ext[2] = {cols, rows}, str[1] = {ld};
    const int box[2] = {kBK, box_rows};
    return capi_encode(m, p, 2, ext, str, box, true, what);
  }

  // The columns as (64, cols / 64) when that divides, so that one box holds
  // two 64-column atoms; else boxes of one atom.
  bool wide() const { return cols % 64 == 0; }

  // 64 rows x 128 columns of one matrix (load_columns).
  int encode_columns(CUtensorMap* m, const char* what) const {
    const int64_t ext[3] = {wide() ? 64 : cols, rows, wide() ? cols / 64 : 1}, str[2] = {ld, wide() ? 64 : ld};
    const int box[3] = {64, kBK, wide() ? 2 : 1};
    return capi_encode(m, p, 3, ext, str, box, true, what);
  }

  // A K block of a stacked weight (load_weights); kmaj: stored N x K.
  int encode_weights(CUtensorMap* m, bool kmaj, const char* what) const {
    // with one matrix the stride is never used, but has to be a legal one
    const int64_t last = batch == 1 ? round_up(rows * ld, 8) : stride;
    const bool w = !kmaj && wide();
    const int64_t ext[4] = {w ? 64 : cols, rows, w ? cols / 64 : 1, batch}, str[3] = {ld, w ? 64 : ld, last};
    const int box[4] = {64, kmaj ? kGrpCols : kBK, w ? 2 : 1, 1};
    return capi_encode(m, p, 4, ext, str, box, true, what);
  }
};

bool misaligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 2u != 0; }

int launch_pack_stacks(const PackJobs& jobs, int sms, cudaStream_t stream) {
  if (jobs.count == 0) return GEMM_OK;
  auto most = [&](int per) {
    long long n = 0;
    for (int j = 0; j < jobs.count; ++j) n = std::max(n, pack_slabs(jobs.job[j], kPackThreads * per) * jobs.job[j].batch);
    return n;
  };
  const bool four = most(4) >= 2 * sms;
  const long long slabs = most(four ? 4 : 1);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<long long>(slabs, 8 * sms)), 1, 1);
  cfg.blockDim = dim3(kPackThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, four ? pack_stacks<4> : pack_stacks<1>, jobs);
  return e == cudaSuccess ? GEMM_OK : capi_fail_cuda(e, "pack_stacks launch");
}

int check_workspace(size_t need, const void* ws, size_t ws_bytes) {
  if (need == 0) return GEMM_OK;
  if (ws == nullptr || ws_bytes < need) {
    return capi_fail(GEMM_ERR_WORKSPACE, "workspace of " + std::to_string(need) + " bytes required, got " +
                                             std::to_string(ws == nullptr ? 0 : ws_bytes));
  }
  if (reinterpret_cast<uintptr_t>(ws) % 256u != 0) {
    return capi_fail(GEMM_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  }
  return GEMM_OK;
}

int check_common(int64_t T, int64_t N, int64_t K, int64_t E, int offsets_bits, int dtype, const char* groups) {
  if (T < 0 || N < 0 || K < 0) return capi_fail(GEMM_ERR_INVALID_ARG, "T, N, K must be >= 0");
  if (T > kMaxExtent || N > kMaxExtent || K > kMaxExtent) {
    return capi_fail(GEMM_ERR_UNSUPPORTED, "T, N, K must each be at most 2^31 - 1024");
  }
  if (E < 1) return capi_fail(GEMM_ERR_INVALID_ARG, std::string(groups) + " must be >= 1");
  if (offsets_bits != 32 && offsets_bits != 64) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "index width must be 32 or 64 bits");
  }
  if (dtype != GEMM_DTYPE_F16 && dtype != GEMM_DTYPE_BF16) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "dtype must be GEMM_DTYPE_F16 or GEMM_DTYPE_BF16");
  }
  return GEMM_OK;
}

// Dynamic shared memory above 48 KiB is opted into once per kernel and device.
template <class Kernel>
cudaError_t opt_in(Kernel kernel, int bytes, std::atomic<unsigned long long>& configured) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (configured.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) configured.fetch_or(bit, std::memory_order_acq_rel);
  return e;
}

// How many clusters of `cluster` CTAs of this kernel the device holds at once
// (GPCs whose SMs do not divide leave some out: a B200 holds 33 of 4 and 15
// of 8 CTAs that fill their SM).  Asked once per kernel, device and size.
template <auto kernel>
int resident_clusters(int bytes, int cluster, int* out) {
  static std::atomic<int> known[64][9];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return capi_fail_cuda(e, "cudaGetDevice");
  std::atomic<int>& slot = known[dev & 63][cluster];
  *out = slot.load(std::memory_order_relaxed);
  if (*out > 0) return GEMM_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(cluster), 1, 1);
  cfg.blockDim = dim3(kGrpThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaOccupancyMaxActiveClusters(out, kernel, &cfg);
  if (e != cudaSuccess) return capi_fail_cuda(e, "cudaOccupancyMaxActiveClusters");
  slot.store(*out, std::memory_order_relaxed);
  return GEMM_OK;
}

template <class Kernel, class... Args>
cudaError_t launch(Kernel kernel, int threads, int bytes, int grid, int cluster, cudaStream_t stream,
                   const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
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
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// `up` is null without adapters.
template <int CG, int TM, int STAGES, bool LORA>
int launch_grouped(const Operand& a, const Operand& b, const Operand* up, const GroupedParams& gp, int sms,
                   cudaStream_t stream) {
  using Plan = GroupedPlan<CG, TM, STAGES, LORA>;
  GroupedParams p = gp;
  p.tiles_n = static_cast<int>((static_cast<int64_t>(p.N) + kGrpCols * CG - 1) / (kGrpCols * CG));
  // the most row tiles that T rows in E groups can make
  const int64_t row_tiles = std::min<int64_t>(p.T, (static_cast<int64_t>(p.T) + static_cast<int64_t>(p.E) * (TM - 1)) / TM);
  const int64_t tiles = row_tiles * p.tiles_n;
  if (tiles > kInt32Max) return capi_fail(GEMM_ERR_UNSUPPORTED, "too many output tiles");
  GroupedMaps maps;
  std::memset(&maps, 0, sizeof(maps));
  int st = GEMM_OK;
  if (p.K > 0) {
    const int64_t most = std::min<int64_t>(round_up(p.T, Plan::kStep), Plan::kSubRows) / CG;   // rows of a CTA
    while (p.first_box + 1 < box_count(TM) && most <= box_rows(TM, p.first_box + 1)) ++p.first_box;
    for (int i = p.first_box; i < box_count(TM) && st == GEMM_OK; ++i) {
      st = a.encode_rows(&maps.a[i], box_rows(TM, i), "A");
    }
    if (st == GEMM_OK) st = b.encode_weights(&maps.b, p.b_kmaj != 0, "B");
    p.b_wide = b.wide();
  }
  if (LORA && st == GEMM_OK) {
    st = up->encode_weights(&maps.u, p.up_kmaj != 0, "up");
    p.up_wide = up->wide();
  }
  if (p.c_tma && st == GEMM_OK) {
    const int64_t ext[2] = {p.N, p.T}, str[1] = {p.ldc};
    const int box[2] = {kGrpCols, kGrpChunk};
    st = capi_encode(&maps.c, p.C, 2, ext, str, box, false, "C");
  }
  if (st != GEMM_OK) return st;
  static std::atomic<unsigned long long> configured{0};
  cudaError_t e = opt_in(gemm_grouped_sm100<CG, TM, STAGES, LORA>, Plan::kDynamicBytes, configured);
  if (e != cudaSuccess) return capi_fail_cuda(e, "grouped gemm kernel attribute");
  // Single CTAs: the cluster that splits the K of the last tiles, at least 8 K
  // blocks to a CTA.  Four or eight CTAs while there is a cluster for every
  // tile; two otherwise.  The number of tiles is an upper bound: only the
  // device knows the groups.
  int cluster = CG;
  if (CG == 1 && p.kb_total >= 16) {
    cluster = 2;
    for (int c = 4; c <= 8 && p.kb_total >= 8 * c; c *= 2) {
      int fit = 0;
      st = resident_clusters<gemm_grouped_sm100<CG, TM, STAGES, LORA>>(Plan::kDynamicBytes, c, &fit);
      if (st != GEMM_OK) return st;
      if (tiles > fit) break;
      cluster = c;
    }
  }
  // persistent: at most one CTA per SM
  const int grid = static_cast<int>(std::min<int64_t>(tiles * Plan::kSubs, sms / cluster)) * cluster;
  e = launch(gemm_grouped_sm100<CG, TM, STAGES, LORA>, kGrpThreads, Plan::kDynamicBytes, grid, cluster,
             stream, maps, p);
  return e == cudaSuccess ? GEMM_OK : capi_fail_cuda(e, "grouped gemm kernel launch");
}

// ------------------------------------------------------------- low-rank adapters
// Workspace of a call with adapters: h, then repacked operands.
struct LoraPlan {
  Operand x, w, up;
  size_t off_h = 0, total = 0;

  LoraPlan(const void* X, const void* W, const void* U, int64_t T, int64_t N, int64_t K, int64_t L, int64_t R,
           int64_t ldx, int64_t ldw, int trans_w, int64_t ld_up, int64_t stride_up, int trans_up)
      : x(X, 1, T, K, ldx, 0), w(W, 1, trans_w ? N : K, trans_w ? K : N, ldw, 0),
        up(U, L, trans_up ? N : R, trans_up ? R : N, ld_up, stride_up) {
    size_t off = align256(gemm_workspace_counter_bytes());
    off_h = off;
    off = align256(off + static_cast<size_t>(T) * shrink_pitch(R) * sizeof(float));
    x.plan(&off);
    w.plan(&off);
    up.plan(&off);
    total = off;
  }
};

constexpr int kWgradStages = 4;

int launch_wgrad(const Operand& a, const Operand& g, const WgradParams& wp, int sms, cudaStream_t stream) {
  using Plan = WgradPlan<kWgradStages>;
  WgradParams p = wp;
  CUtensorMap tmA, tmG, tmD;
  std::memset(&tmD, 0, sizeof(tmD));
  int st = a.encode_columns(&tmA, "A");
  if (st == GEMM_OK) st = g.encode_columns(&tmG, "G");
  p.a_wide = a.wide();
  p.g_wide = g.wide();
  if (st != GEMM_OK) return st;
  if (p.d_tma) {
    const int64_t ext[3] = {p.N, p.M, p.E}, str[2] = {p.ldd, p.E == 1 ? round_up(p.M * p.ldd, 8) : p.stride_d};
    const int box[3] = {kStoreCols, kStoreRows, 1};
    st = capi_encode(&tmD, p.D, 3, ext, str, box, true, "D");
    if (st != GEMM_OK) return st;
  }
  const int64_t tiles = static_cast<int64_t>(p.E) * p.tiles_m * p.tiles_n;
  const int grid = static_cast<int>(std::min<int64_t>(tiles, sms / 2)) * 2;
  static std::atomic<unsigned long long> configured{0};
  cudaError_t e = opt_in(gemm_grouped_wgrad_sm100<kWgradStages>, Plan::kDynamicBytes, configured);
  if (e != cudaSuccess) return capi_fail_cuda(e, "grouped weight gradient kernel attribute");
  e = launch(gemm_grouped_wgrad_sm100<kWgradStages>, kWgradThreads, Plan::kDynamicBytes, grid, 2, stream, tmA, tmG, tmD,
             p);
  return e == cudaSuccess ? GEMM_OK : capi_fail_cuda(e, "grouped weight gradient kernel launch");
}

// Single CTAs of 128 columns x up to 64 rows, or pairs of 256 x up to 256?
//  * Up to 16 rows per group: the cost is reading the weights once, and single
//    CTAs with their deep ring do that best (32 rows over 64 experts 2048 x
//    1024: 25 us against 29).
//  * More rows: pairs, which read every weight once per 256 rows (4096 rows
//    over 64 experts 2048 x 1024: 55 us against 68), unless their tiles would
//    leave more than half of the machine idle where single CTAs fill it
//    (64 rows, 4096 x 4096: 32 clusters of 4 in 13 us against 16 pairs in 26).
bool small_tiles(int64_t T, int64_t N, int64_t E, int sms) {
  if (T <= 16 * E || N <= kGrpCols) return true;
  const int64_t pairs = (T + 255 * E) / 256 * ((N + 255) / 256);
  const int64_t singles = (T + 63 * E) / 64 * ((N + 127) / 128);
  return 4 * pairs < sms && singles <= sms;
}

// Pair tiles of 512 rows instead of 256?  They read a quarter less from L2 per
// product, but their epilogue is not hidden and a short last wave costs more:
// for groups of 1024 rows and more on average and three waves at least.
// Under the power cap, 8192 rows over 8 experts 4096 x 14336: 769 us against
// 812 (ragged groups 811 against 852), 4096 x 4096: 223 against 230.  Below:
// 2048 rows over 2 experts 4096 x 4096 70 us against 57, 4096 rows over 8
// experts 4096 x 14336 458 us against 427.  (Both columns are medians of calls
// back to back; the first pair of lines after a second of them.)
bool tall_tiles(int64_t T, int64_t N, int64_t E, int sms) {
  return T >= 1024 * E && T / 512 * ((N + 255) / 256) >= 3 * (sms / 2);
}

Operand operand_b(const void* B, int64_t E, int64_t N, int64_t K, int64_t ldb, int64_t stride_b, int trans_b) {
  return Operand(B, E, trans_b ? N : K, trans_b ? K : N, ldb, stride_b);
}

}  // namespace
}  // namespace idb

using namespace idb;

extern "C" {

size_t gemm_grouped_workspace_bytes(const void* A, const void* B, int64_t T, int64_t N, int64_t K, int64_t E,
                                    int64_t lda, int64_t ldb, int64_t stride_b, int trans_b) {
  if (T <= 0 || N <= 0 || K < 0 || E < 1) return 0;
  Operand a(A, 1, T, K, lda, 0), b = operand_b(B, E, N, K, ldb, stride_b, trans_b);
  const size_t head = align256(gemm_workspace_counter_bytes());
  size_t off = head;
  a.plan(&off);
  b.plan(&off);
  return off == head ? 0 : off;
}

int gemm_grouped_launch(const void* A, const void* B, void* C, const void* offsets, int offsets_bits, int64_t T,
                        int64_t N, int64_t K, int64_t E, int64_t lda, int64_t ldb, int64_t stride_b, int64_t ldc,
                        int trans_b, const void* bias, int activation, int zero_rest, int dtype, void* workspace,
                        size_t workspace_bytes, void* stream_v) {
  capi_clear_error();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  int st = check_common(T, N, K, E, offsets_bits, dtype, "the number of groups");
  if (st != GEMM_OK) return st;
  if (E > kMaxGroups) {
    return capi_fail(GEMM_ERR_UNSUPPORTED, "at most " + std::to_string(kMaxGroups) + " groups");
  }
  if (trans_b != 0 && trans_b != 1) return capi_fail(GEMM_ERR_INVALID_ARG, "trans_b must be 0 or 1");
  if (activation < GEMM_ACT_NONE || activation > GEMM_ACT_GELU) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "activation must be GEMM_ACT_NONE, GEMM_ACT_RELU or GEMM_ACT_GELU");
  }
  if (T == 0 || N == 0) return GEMM_OK;
  if (!C || !offsets || (K > 0 && (!A || !B))) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "A, B, C and offsets must be non-null");
  }
  const int64_t b_rows = trans_b ? N : K, b_cols = trans_b ? K : N;
  if (lda < K || ldb < b_cols || ldc < N || (E > 1 && b_rows > 0 && stride_b < (b_rows - 1) * ldb + b_cols)) {
    return capi_fail(GEMM_ERR_INVALID_ARG, std::string("pitches must satisfy lda >= K, ldb >= ") +
                                               (trans_b ? "K" : "N") + ", ldc >= N, and stride_b one matrix of B");
  }
  if (misaligned(A) || misaligned(B) || misaligned(C) || misaligned(bias)) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "A, B, C and bias must be 2-byte aligned");
  }
  if (reinterpret_cast<uintptr_t>(offsets) % (offsets_bits / 8) != 0) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "offsets must be aligned to their width");
  }
  Operand a(A, 1, T, K, lda, 0), b = operand_b(B, E, N, K, ldb, stride_b, trans_b);
  const size_t head = align256(gemm_workspace_counter_bytes());
  size_t off = head;
  a.plan(&off);
  b.plan(&off);
  st = check_workspace(off == head ? 0 : off, workspace, workspace_bytes);
  if (st != GEMM_OK) return st;

  GroupedParams p = {};
  int sms = 0;
  st = capi_device(&sms, &p.err);
  if (st != GEMM_OK) return st;
  PackJobs jobs = {};
  a.add(static_cast<uint8_t*>(workspace), &jobs);
  b.add(static_cast<uint8_t*>(workspace), &jobs, offsets, offsets_bits == 64);
  st = launch_pack_stacks(jobs, sms, stream);
  if (st != GEMM_OK) return st;
  p.offsets = offsets;
  p.off64 = offsets_bits == 64;
  p.E = static_cast<int>(E);
  p.T = static_cast<int>(T);
  p.N = static_cast<int>(N);
  p.K = static_cast<int>(K);
  p.kb_total = static_cast<int>((K + kBK - 1) / kBK);
  p.b_kmaj = trans_b;
  p.bf16 = dtype == GEMM_DTYPE_BF16;
  p.act = activation;
  p.bias = static_cast<const unsigned short*>(bias);
  p.C = static_cast<unsigned short*>(C);
  p.ldc = ldc;
  p.c_tma = p.c_vec = reinterpret_cast<uintptr_t>(C) % 16u == 0 && ldc % 8 == 0;
  p.zero_rest = zero_rest != 0;
  if (small_tiles(T, N, E, sms)) return launch_grouped<1, 64, 7, false>(a, b, nullptr, p, sms, stream);
  if (tall_tiles(T, N, E, sms)) return launch_grouped<2, 512, 4, false>(a, b, nullptr, p, sms, stream);
  return launch_grouped<2, 256, 6, false>(a, b, nullptr, p, sms, stream);
}

size_t gemm_grouped_wgrad_workspace_bytes(const void* A, const void* G, int64_t T, int64_t M, int64_t N, int64_t lda,
                                          int64_t ldg) {
  if (T <= 0 || M <= 0 || N <= 0) return 0;
  Operand a(A, 1, T, M, lda, 0), g(G, 1, T, N, ldg, 0);
  const size_t head = align256(gemm_workspace_counter_bytes());
  size_t off = head;
  a.plan(&off);
  g.plan(&off);
  return off == head ? 0 : off;
}

int gemm_grouped_wgrad_launch(const void* A, const void* G, void* D, const void* offsets, int offsets_bits, int64_t T,
                              int64_t M, int64_t N, int64_t E, int64_t lda, int64_t ldg, int64_t ldd, int64_t stride_d,
                              int dtype, void* workspace, size_t workspace_bytes, void* stream_v) {
  capi_clear_error();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  int st = check_common(T, N, M, E, offsets_bits, dtype, "the number of groups");
  if (st != GEMM_OK) return st;
  if (E > kMaxGroups) {
    return capi_fail(GEMM_ERR_UNSUPPORTED, "at most " + std::to_string(kMaxGroups) + " groups");
  }
  if (M == 0 || N == 0) return GEMM_OK;
  if (!D || (T > 0 && (!A || !G || !offsets))) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "A, G, D and offsets must be non-null");
  }
  if ((T > 0 && (lda < M || ldg < N)) || ldd < N || (E > 1 && stride_d < (M - 1) * ldd + N)) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "pitches must satisfy lda >= M, ldg >= N, ldd >= N, and stride_d one "
                                           "matrix of D");
  }
  if (misaligned(A) || misaligned(G) || misaligned(D)) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "A, G and D must be 2-byte aligned");
  }
  if (reinterpret_cast<uintptr_t>(offsets) % (offsets_bits / 8) != 0) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "offsets must be aligned to their width");
  }
  WgradParams p = {};
  const int64_t tm = (M + kWgradTile - 1) / kWgradTile, tn = (N + kWgradTile - 1) / kWgradTile;
  if (tm * tn > kInt32Max / E) return capi_fail(GEMM_ERR_UNSUPPORTED, "too many output tiles");
  Operand a(A, 1, T, M, lda, 0), g(G, 1, T, N, ldg, 0);
  const size_t head = align256(gemm_workspace_counter_bytes());
  size_t off = head;
  a.plan(&off);
  g.plan(&off);
  st = check_workspace(off == head ? 0 : off, workspace, workspace_bytes);
  if (st != GEMM_OK) return st;
  int sms = 0;
  st = capi_device(&sms, &p.err);
  if (st != GEMM_OK) return st;
  if (T == 0) {   // no rows: every gradient is zero
    for (int64_t e = 0; e < E; ++e) {
      cudaError_t ce = cudaMemset2DAsync(static_cast<uint8_t*>(D) + e * stride_d * 2, static_cast<size_t>(ldd) * 2, 0,
                                         static_cast<size_t>(N) * 2, static_cast<size_t>(M), stream);
      if (ce != cudaSuccess) return capi_fail_cuda(ce, "cudaMemset2DAsync");
    }
    return GEMM_OK;
  }
  PackJobs jobs = {};
  a.add(static_cast<uint8_t*>(workspace), &jobs);
  g.add(static_cast<uint8_t*>(workspace), &jobs);
  st = launch_pack_stacks(jobs, sms, stream);
  if (st != GEMM_OK) return st;
  p.offsets = offsets;
  p.off64 = offsets_bits == 64;
  p.E = static_cast<int>(E);
  p.T = static_cast<int>(T);
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.tiles_m = static_cast<int>(tm);
  p.tiles_n = static_cast<int>(tn);
  p.bf16 = dtype == GEMM_DTYPE_BF16;
  p.D = static_cast<unsigned short*>(D);
  p.ldd = ldd;
  p.stride_d = E == 1 ? 0 : stride_d;
  p.d_tma = reinterpret_cast<uintptr_t>(D) % 16u == 0 && ldd % 8 == 0 && (E == 1 || stride_d % 8 == 0);
  return launch_wgrad(a, g, p, sms, stream);
}

size_t gemm_lora_workspace_bytes(const void* X, const void* W, const void* up, int64_t T, int64_t N, int64_t K,
                                 int64_t L, int64_t R, int64_t ldx, int64_t ldw, int trans_w, int64_t ld_up,
                                 int64_t stride_up, int trans_up) {
  if (T <= 0 || N <= 0 || K <= 0 || L <= 0 || R <= 0) return 0;
  return LoraPlan(X, W, up, T, N, K, L, R, ldx, ldw, trans_w, ld_up, stride_up, trans_up).total;
}

int gemm_lora_launch(const void* X, const void* W, const void* down, const void* up, void* C, const void* adapter,
                     int adapter_bits, int64_t T, int64_t N, int64_t K, int64_t L, int64_t R, int64_t ldx, int64_t ldw,
                     int trans_w, int64_t ld_down, int64_t stride_down, int trans_down, int64_t ld_up,
                     int64_t stride_up, int trans_up, int64_t ldc, const float* scale, const void* bias, int activation,
                     int dtype, void* workspace, size_t workspace_bytes, void* stream_v) {
  capi_clear_error();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  int st = check_common(T, N, K, L, adapter_bits, dtype, "the number of adapters");
  if (st != GEMM_OK) return st;
  if (K < 1) return capi_fail(GEMM_ERR_INVALID_ARG, "K must be >= 1");
  if (R < 1 || R > GEMM_LORA_MAX_RANK) {
    return capi_fail(R < 1 ? GEMM_ERR_INVALID_ARG : GEMM_ERR_UNSUPPORTED,
                     "the rank must be in [1, " + std::to_string(GEMM_LORA_MAX_RANK) + "]");
  }
  if (L > kInt32Max) return capi_fail(GEMM_ERR_UNSUPPORTED, "the number of adapters must be < 2^31");
  if ((trans_w != 0 && trans_w != 1) || (trans_down != 0 && trans_down != 1) || (trans_up != 0 && trans_up != 1)) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "trans_w, trans_down and trans_up must be 0 or 1");
  }
  if (activation < GEMM_ACT_NONE || activation > GEMM_ACT_GELU) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "activation must be GEMM_ACT_NONE, GEMM_ACT_RELU or GEMM_ACT_GELU");
  }
  if (T == 0 || N == 0) return GEMM_OK;
  if (!X || !W || !down || !up || !C || !adapter) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "X, W, down, up, C and adapter must be non-null");
  }
  const int64_t down_rows = trans_down ? R : K, down_cols = trans_down ? K : R;
  const int64_t up_rows = trans_up ? N : R, up_cols = trans_up ? R : N;
  if (ldx < K || ldw < (trans_w ? K : N) || ldc < N || ld_down < down_cols || ld_up < up_cols ||
      (L > 1 && (stride_down < (down_rows - 1) * ld_down + down_cols || stride_up < (up_rows - 1) * ld_up + up_cols))) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "a pitch is shorter than its row, or a stride than its matrix");
  }
  if (misaligned(X) || misaligned(W) || misaligned(down) || misaligned(up) || misaligned(C) || misaligned(bias)) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "X, W, down, up, C and bias must be 2-byte aligned");
  }
  if (reinterpret_cast<uintptr_t>(adapter) % (adapter_bits / 8) != 0 || reinterpret_cast<uintptr_t>(scale) % 4u != 0) {
    return capi_fail(GEMM_ERR_INVALID_ARG, "adapter and scale must be aligned to their width");
  }
  LoraPlan pl(X, W, up, T, N, K, L, R, ldx, ldw, trans_w, ld_up, stride_up, trans_up);
  st = check_workspace(pl.total, workspace, workspace_bytes);
  if (st != GEMM_OK) return st;
  GroupedParams p = {};
  int sms = 0;
  st = capi_device(&sms, &p.err);
  if (st != GEMM_OK) return st;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  PackJobs jobs = {};
  pl.x.add(ws, &jobs);
  pl.w.add(ws, &jobs);
  pl.up.add(ws, &jobs);
  st = launch_pack_stacks(jobs, sms, stream);
  if (st != GEMM_OK) return st;

  ShrinkParams s = {};
  s.x = static_cast<const unsigned short*>(pl.x.p);
  s.ldx = pl.x.ld;
  s.down = static_cast<const unsigned short*>(down);
  s.ld_down = ld_down;
  s.stride_down = L == 1 ? 0 : stride_down;
  s.adapter = adapter;
  s.adapter64 = adapter_bits == 64;
  s.scale = scale;
  s.h = reinterpret_cast<float*>(ws + pl.off_h);
  s.h_pitch = static_cast<int>(shrink_pitch(R));
  s.T = static_cast<int>(T);
  s.K = static_cast<int>(K);
  s.L = static_cast<int>(L);
  s.R = static_cast<int>(R);
  s.err = p.err;
  st = launch_shrink(s, trans_down != 0, dtype == GEMM_DTYPE_BF16, sms, stream);   // x is TMA-addressable by now
  if (st != GEMM_OK) return st;

  p.E = 1;
  p.T = s.T;
  p.N = static_cast<int>(N);
  p.K = s.K;
  p.kb_total = static_cast<int>((K + kBK - 1) / kBK);
  p.b_kmaj = trans_w;
  p.bf16 = dtype == GEMM_DTYPE_BF16;
  p.act = activation;
  p.bias = static_cast<const unsigned short*>(bias);
  p.C = static_cast<unsigned short*>(C);
  p.ldc = ldc;
  p.c_tma = p.c_vec = reinterpret_cast<uintptr_t>(C) % 16u == 0 && ldc % 8 == 0;
  p.h = s.h;
  p.h_pitch = s.h_pitch;
  p.L = s.L;
  p.R = s.R;
  p.adapter = adapter;
  p.adapter64 = s.adapter64;
  p.up_kmaj = trans_up;
  p.up = static_cast<const unsigned short*>(pl.up.p);
  p.ld_up = pl.up.ld;
  p.stride_up = L == 1 ? 0 : pl.up.stride;
  p.packed = jobs.count > 0;
  if (small_tiles(T, N, 1, sms)) return launch_grouped<1, 64, 6, true>(pl.x, pl.w, &pl.up, p, sms, stream);
  return launch_grouped<2, 256, 6, true>(pl.x, pl.w, &pl.up, p, sms, stream);
}

}  // extern "C"
