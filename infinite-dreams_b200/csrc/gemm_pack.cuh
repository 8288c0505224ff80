// Repacking of 16-bit rows whose base or pitch TMA cannot address.
#pragma once
#include "sm100_ptx.cuh"

namespace idb {

// Bytes o .. o + 15 (o even) of the 32 bytes c0, c1: the words are shifted
// into place in registers, in 8-, 4- and 2-byte steps.
__device__ __forceinline__ uint4 shift_chunks(uint4 c0, uint4 c1, int o) {
  uint32_t w0 = c0.x, w1 = c0.y, w2 = c0.z, w3 = c0.w, w4 = c1.x, w5 = c1.y, w6 = c1.z, w7 = c1.w;
  if (o & 8) {
    w0 = w2; w1 = w3; w2 = w4; w3 = w5; w4 = w6; w5 = w7;
  }
  if (o & 4) {
    w0 = w1; w1 = w2; w2 = w3; w3 = w4; w4 = w5;
  }
  if (o & 2) {  // bytes 2..3 of one word, then bytes 0..1 of the next
    w0 = __byte_perm(w0, w1, 0x5432);
    w1 = __byte_perm(w1, w2, 0x5432);
    w2 = __byte_perm(w2, w3, 0x5432);
    w3 = __byte_perm(w3, w4, 0x5432);
  }
  return make_uint4(w0, w1, w2, w3);
}

// The 8 elements at the 2-byte aligned address `a`, of which the first `left`
// belong to the row (the others read as zero), out of a matrix in [begin,
// end).  The one or two aligned 16-byte chunks that cover them are read with
// vector loads (neighbouring threads read the same chunks, which the cache
// serves); what they hold of the next row is masked.  Where such a chunk would
// reach outside the matrix the elements are read one by one, so no load leaves
// the caller's memory.
__device__ __forceinline__ uint4 pack_chunk(uintptr_t begin, uintptr_t end, uintptr_t a, int left) {
  const uintptr_t lo = a & ~static_cast<uintptr_t>(15);
  const int o = static_cast<int>(a - lo);
  if (lo >= begin && lo + (o ? 32u : 16u) <= end) {
    uint4 v = __ldg(reinterpret_cast<const uint4*>(lo));
    if (o) v = shift_chunks(v, __ldg(reinterpret_cast<const uint4*>(lo + 16)), o);
    if (left < 8) {
      auto keep = [&](uint32_t w, int i) { return left > i + 1 ? w : (left > i ? w & 0xFFFFu : 0u); };
      v = make_uint4(keep(v.x, 0), keep(v.y, 2), keep(v.z, 4), keep(v.w, 6));
    }
    return v;
  }
  const unsigned short* sp = reinterpret_cast<const unsigned short*>(a);
  unsigned short v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (i < left) ? sp[i] : static_cast<unsigned short>(0);
  return make_uint4(v[0] | (static_cast<unsigned>(v[1]) << 16), v[2] | (static_cast<unsigned>(v[3]) << 16),
                    v[4] | (static_cast<unsigned>(v[5]) << 16), v[6] | (static_cast<unsigned>(v[7]) << 16));
}

// Several stacks of matrices in one launch.
struct PackJob {
  const void* src;       // `batch` matrices of rows x cols, pitch lds, `stride` elements apart
  long long lds, stride;
  void* dst;             // one matrix after the other, pitch ldd
  long long ldd;
  int batch, rows, cols;
  const void* offsets;   // not null: matrix b is skipped unless offsets[b] < offsets[b + 1]
  int off64;
};
constexpr int kMaxPackJobs = 3;
struct PackJobs {
  PackJob job[kMaxPackJobs];
  int count;
};

}  // namespace idb
