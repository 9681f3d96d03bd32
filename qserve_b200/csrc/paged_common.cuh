// qserve_b200 -- what the operators over portions of sequences in the paged key/value cache share (paged_cache.cu, paged_attention.cu).
//
// A page holds 64 positions of all kv heads: codes [Hkv][64][128 * BITS / 8] | scales fp16 [Hkv][64] | zeros fp16 [Hkv][64].  INT4: the even element of a byte
// in its low nibble.  Code u of a row with scale s and zero z stands for s u + half(-s z) (INT4), s (u - z) (INT8).
#pragma once
#include "common.cuh"
#include "launch.h"

namespace qs {
namespace paged {

constexpr int kD = 128;    // head size
constexpr int kPage = 64;  // positions of a page

template <int BITS>
struct Geom {
  static constexpr int kRow = kD * BITS / 8;      // bytes of codes of a position of one head
  static constexpr int kCodes = kPage * kRow;     // bytes of codes of one head of a page
  static __host__ __device__ long long codes_at(int head) { return static_cast<long long>(head) * kCodes; }
  static __host__ __device__ long long scales_at(int head, int kv_heads) { return static_cast<long long>(kv_heads) * kCodes + head * (kPage * 2); }
  static __host__ __device__ long long zeros_at(int head, int kv_heads) { return scales_at(head, kv_heads) + kv_heads * (kPage * 2); }
};

__device__ __forceinline__ uint32_t lop3_and_or(uint32_t x, uint32_t mask, uint32_t orv) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(x), "r"(mask), "r"(orv));  // (x & mask) | orv
  return d;
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// Codes as fp16 numbers, exactly: 0x6400 | u is 1024 + u, 0x6400 | 16 u is 1024 + 16 u.
// INT4: the eight codes of a word as (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ void codes_of_word4(uint32_t w, __half2 (&u)[4]) {
  const __half2 low = __float2half2_rn(-1024.f), sixteenth = __float2half2_rn(0.0625f), high = __float2half2_rn(-64.f);
  const uint32_t t = w >> 8;
  u[0] = __hadd2(as_h2(lop3_and_or(w, 0x000f000fu, 0x64006400u)), low);
  u[1] = __hfma2(as_h2(lop3_and_or(w, 0x00f000f0u, 0x64006400u)), sixteenth, high);
  u[2] = __hadd2(as_h2(lop3_and_or(t, 0x000f000fu, 0x64006400u)), low);
  u[3] = __hfma2(as_h2(lop3_and_or(t, 0x00f000f0u, 0x64006400u)), sixteenth, high);
}
// INT8: the four codes of a word as (0, 1), (2, 3), each plus 1024 + low: exact for whole numbers low from -2048 to 0
__device__ __forceinline__ void codes_of_word8(uint32_t w, __half2 low, __half2 (&u)[2]) {
  u[0] = __hadd2(as_h2(__byte_perm(w, 0x64006400u, 0x7150)), low);
  u[1] = __hadd2(as_h2(__byte_perm(w, 0x64006400u, 0x7352)), low);
}

// What a batch of portions says about one of its sequences: `first` the position of its first new token, `start` that token's row.  Whatever the tables say,
// rows stay inside the batch's.
struct Portion {
  int start, count, first;
};
__device__ __forceinline__ Portion portion_of(const int* cu, const int* lengths, int b, int num_tokens) {
  Portion p;
  const int lo = cu ? cu[b] : b, hi = cu ? cu[b + 1] : b + 1;
  p.start = min(max(lo, 0), num_tokens);
  p.count = max(min(hi, num_tokens) - p.start, 0);
  p.first = min(max(lengths[b], 0), 1 << 30) - min(max(hi - lo, 0), 1 << 30);  // (within 31 bits whatever the tables say)
  return p;
}
// all lanes of a warp: the sequence that row t belongs to, -1 behind the last one (cu ascending)
__device__ __forceinline__ int sequence_of(const int* cu, int batch, int t) {
  if (!cu) return t < batch ? t : -1;
  const int lane = threadIdx.x & 31;
  int below = 0;  // how many sequences start at t or ahead of it
  for (int i = 0; i <= batch; i += 32) below += __popc(__ballot_sync(0xffffffffu, i + lane <= batch && cu[i + lane] <= t));
  return below >= 1 && below <= batch ? below - 1 : -1;
}

template <typename Kern, typename... Args>
int launch(Kern kern, dim3 grid, int threads, size_t smem, void* stream, const char* what, int cluster, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, args...), what);
}

}  // namespace paged
}  // namespace qs
