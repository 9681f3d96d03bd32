// qserve_b200 -- attention over the paged INT4 / INT8 cache of many query rows per key: portions of prompts (qs_paged_prompt_attention), and single tokens of a
// batch whose sequences share their first pages (qs_shared_prefix_attention).
//
// Tile kernel.  The rows of a tile are (token, query head) pairs of one kv head: 128 rows see the same keys, whose codes are unpacked once for all of them.  Per
// page of 64 keys:
//     unpack          4 warps: codes, scales and zeros (one tile: from registers that they load a page ahead; two: from a ring of raw slots that bulk copies
//                     fill) -> fp16 numbers in the swizzled shared-memory form that the products take (keys past the last row's limit: zeros)
//     S = Q K^T       8 x tcgen05.mma 128 x 64 x 16, accumulators in tensor memory
//     softmax         4 warps, thread = row (tensor memory lane): running maximum and sum in 32 bits, P = exp2(..) rounded to fp16, into tensor memory
//     O += P V        4 x tcgen05.mma 128 x 128 x 16, A from tensor memory
// fp16 holds the operands (keys, values and weights, each off by 2^-11 of itself at most, INT8 keys and values by another 2^-12 of their scale): a product of exact
// codes would want every score multiplied by its key's scale and every weight by its value's, a third more instructions of softmax warps that are the bound already.
// A result is off by 4.2e-4 to 4.7e-4 so, where its own rounding alone is 2.1e-4.
// A long axis of keys is split over blocks where the rows alone do not fill the device, or not its last round.  A split leaves its rows' maximum, sum and O / sum in
// fp32; the cluster that holds all splits, join_kernel (prompts) or the tail kernel (shared prefix) joins them.  (O / sum in fp16 would be one more rounding of a
// result and half the bytes; us, fp16 / now: 17 tokens behind 500 7.8 / 8.4, 24 behind 60000 41.8 / 43.4, 8 sequences behind 1024 shared positions 8.0 / 8.4, 64
// behind 8192 30.3 / 31.6.)
// Bounds: 4096 tokens of 32 heads over 8 behind 12000 positions, INT4, 798 us at 1965 MHz (0.94 TFLOP, 1.18 PFLOP/s; 870 to 920 in runs
// of seconds, where the power limit leaves 1.67 GHz), shared memory 0.88 of its cycles (the queries are read again for every 64 keys, unpacked pages written and read)
// and issue slots 0.54, the tensor pipe 0.60; one tile: the chain load - unpack - softmax of a page,
// 0.85 us with two blocks per multiprocessor.
//
// Tail kernel (shared prefix): the pages behind the shared ones (all pages, for few sequences) on mma.sync, eight query heads a product, codes taken as they lie.  A
// cluster of blocks per (sequence, run of heads) that deals the pages out to its warps, or, for batches that fill the device that way, a warp each; joins its warps',
// its cluster's and the prefix's partial rows and writes the result.  200 sequences of 2000 positions, 8 kv heads, INT4: 78 us, prefix of a page and all, for 328 MB.
#include <math_constants.h>

#include <type_traits>

#include "paged_common.cuh"

namespace qs {
namespace {

using namespace paged;

// ------------------------------------------------------------------------------------------------------------------------
// PTX
// ------------------------------------------------------------------------------------------------------------------------
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t m, uint32_t n, uint32_t b_mn_major) {
  // D = f32 (bits 4..5 = 1), A = B = f16, A K-major, B K-major or MN-major (bit 16), N >> 3 at bit 17, M >> 4 at bit 24
  return (1u << 4) | (b_mn_major << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :
      : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();  // the barrier's aligned form is for whole warps, and whoever calls may come out of a branch or loop that lanes left one by one
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// eight bytes at this place of the shared memory of block `rank` of the cluster
__device__ __forceinline__ uint2 peer_u2(const void* mine, uint32_t rank) {
  uint32_t a;
  uint2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ float peer_f32(const float* mine, uint32_t rank) {
  uint32_t a;
  float f;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
  return f;
}
__device__ __forceinline__ float4 peer_f32x4(const float* mine, uint32_t rank) {
  uint32_t a;
  float4 f;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "r"(a) : "memory");
  return f;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// rows of 128 bytes = 64 neighbours along N, one row per K index, 128-byte swizzle; lbo: from one 64-column group to the next, 1024 bytes from 8 K rows to the next 8
__device__ __forceinline__ uint64_t desc_sw128_mn(uint32_t smem_addr, uint32_t lbo_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4);
  d |= static_cast<uint64_t>(lbo_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// ------------------------------------------------------------------------------------------------------------------------
// tile kernel
// ------------------------------------------------------------------------------------------------------------------------
constexpr int kRows = 128;                   // rows of a tile
constexpr int kQBytes = kRows * kD * 2;      // two swizzled halves of 64 columns
constexpr int kKvBytes = kPage * kD * 2;     // a page's K or V as fp16, two halves
constexpr int kKvHalf = kKvBytes / 2;
constexpr int kMostCluster = 8;
constexpr float kRescale = 8.f;              // log2 units that a row's maximum may grow before O is rescaled
constexpr float kLift = 6.f;                 // log2 of the largest weight after that: fp16 holds 2^14, and weights down to 2^-20 of the largest are no subnormal numbers
// Of a tile's tensor memory columns: S and then P of even pages [0, 64), of odd pages [64, 128), O [128, 256).  A page's P takes the place of its own S, so the next
// page's S is there before this one's softmax ends, and P waits for no product.
constexpr uint32_t kTileCols = 256, kColO = 128;

// Registers per thread that the three warpgroups of a one-tile block trade for the launch's 80 (two blocks per multiprocessor): the softmax's increase waits until
// its share is free, for good where the launch brought fewer than all shares together, and a decrease may not name more than there are, so the host asks before
// the first launch.
constexpr int kSoftmaxRegs = 112, kUnpackRegs = 80, kIssueRegs = 48;
constexpr bool shares_suffice(int per_thread) {
  return 3 * per_thread >= kSoftmaxRegs + kUnpackRegs + kIssueRegs && per_thread >= kUnpackRegs && per_thread >= kIssueRegs && per_thread <= kSoftmaxRegs;
}

template <int BITS, int TILES>
struct TileCfg {
  static constexpr bool kShares = TILES == 1;
  static constexpr int kSoftmaxWarps = 4 * TILES;
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 4 + 4);  // softmax, unpack, a warpgroup of which a warp per tile issues products
  static constexpr int kBlocksPerSm = TILES == 1 ? 2 : 1;
  static constexpr int kKStages = 2, kVStages = 2;
  // One tile: the unpacking threads load codes, scales and zeros themselves, a page ahead in registers.  Two: a warp of its own has bulk copies bring them into a ring
  // of raw slots.  us when it was chosen, ring / registers: 17 tokens behind 500 10.5 / 9.3, 8 sequences behind 1024 shared positions 9.8 / 8.3; 4096 tokens behind
  // 12000 852 / 960 (two tiles leave the unpacking threads no time for loads).
  static constexpr bool kRing = TILES == 2;
  static constexpr int kSlots = kRing ? (BITS == 4 ? 8 : 5) : 0;
  static constexpr int kCodes = Geom<BITS>::kCodes;
  static constexpr int kMeta = 2 * kCodes;               // of a slot: codes of K and V, then K scales, K zeros, V scales, V zeros, 128 bytes each
  static constexpr int kSlotBytes = 2 * kCodes + 512;
  static constexpr int kOffK = TILES * kQBytes, kOffV = kOffK + kKStages * kKvBytes, kOffRaw = kOffV + kVStages * kKvBytes;
  static constexpr int kOffBar = kOffRaw + kSlots * kSlotBytes;
  static constexpr int kSmem = kOffBar + 384;
  static_assert(kSmem * kBlocksPerSm + 1024 * kBlocksPerSm <= 228 * 1024, "shared memory of a multiprocessor");
};

struct TileParams {
  const __half* q;
  __half* out;
  long long q_stride, out_stride;
  const long long* kv_pointers;
  const int *cu, *lengths;
  int batch, num_tokens, max_seqlen, max_blocks, num_heads, num_kv_heads;
  int row_blocks, nsplit, shared_blocks;  // shared_blocks > 0: the rows of all sequences over the first sequence's first pages
  int cluster, parts;                     // blocks that join their splits through one another's shared memory; partial rows that are left: nsplit / cluster
  int block_rows, split_from, run;        // of the items (of so many rows each; last rows first, sequence, kv head) those from here on are split; so many neighbours a run
  float scale_log2;
  // parts > 1: O / sum [rows][parts][128]: rows = token * num_heads + head where all items are split, otherwise those of the split items, one behind the other
  float* part;
  float2* part_ml;                        // (maximum, sum) [rows][parts]
};

// Two results in fp16, no further from 0 than its largest number (NaN stays NaN): a mean of values is no larger than they are, but rounded weights over the sum of the
// unrounded ones may be 2^-11 more than 1, and 65504 of that rounds to infinity
__device__ __forceinline__ uint32_t results(float a, float b) {
  uint32_t d;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}
__device__ __forceinline__ uint2 scaled_h4(const float4& a, float L) {
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
  return make_uint2(results(a.x * inv, a.y * inv), results(a.z * inv, a.w * inv));
}

// What a block does with its rows: the result; a partial result where its item is split; or its cluster's, joined first.
enum : int { kWhole = 0, kPartial = 1, kCluster = 2 };
// Which of the splits of which item a block takes: runs of items in turn, all of a run's first splits ahead of its second ones.  (Neighbours are the kv heads of the
// same pages, which lie side by side.)
struct Share {
  unsigned item, split, nsplit;
};
template <int MODE>
__device__ __forceinline__ Share share_of(const TileParams& p, unsigned block) {
  Share s{block, 0, 1};
  if constexpr (MODE == kCluster) {
    s.nsplit = p.cluster;  // a power of two
    s.split = block & (s.nsplit - 1);
    s.item = block / s.nsplit;
  } else if (MODE == kPartial && block >= static_cast<unsigned>(p.split_from)) {
    s.nsplit = p.nsplit;
    const unsigned behind = block - p.split_from, in_turn = behind / static_cast<unsigned>(p.run), run = in_turn / s.nsplit;
    s.split = in_turn - run * s.nsplit;
    s.item = p.split_from + run * p.run + (behind - in_turn * p.run);
  }
  return s;
}
template <int BITS, int TILES, int MODE>
__global__ void __launch_bounds__(TileCfg<BITS, TILES>::kThreads, TileCfg<BITS, TILES>::kBlocksPerSm) tile_kernel(const __grid_constant__ TileParams p) {
  using C = TileCfg<BITS, TILES>;
  using G = Geom<BITS>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* bar_q = bar;             // [2] a tile's queries lie in shared memory
  uint64_t* bar_s = bar + 2;         // [2][2] tile, page parity: S complete
  uint64_t* bar_p = bar + 6;         // [2][2] P written
  // [2][2] O += P V retired.  Two, as for S and P: who waits for a page's product may be one page ahead of it or find the next one's done as well, and a barrier
  // that went through two phases looks as if it had gone through none
  uint64_t* bar_o = bar + 10;
  uint64_t* bar_kfull = bar + 14;                     // [stages] K unpacked
  uint64_t* bar_kfree = bar_kfull + C::kKStages;      // S = Q K^T of all tiles retired
  uint64_t* bar_vfull = bar_kfree + C::kKStages;
  uint64_t* bar_vfree = bar_vfull + C::kVStages;
  uint64_t* bar_raw = bar_vfree + C::kVStages;        // [slots] raw slot landed
  uint64_t* bar_used = bar_raw + C::kSlots;           // [slots] raw slot read
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bar_used + C::kSlots);
  // [128] rows' maximum and sum, for the cluster: over V, at the end.  (Shared memory of their own would leave L1 32 KB less: two blocks' 196 KB are a step of its
  // size.  128 INT8 sequences behind 16384, when it was chosen: 137 us, 158 so)
  float2* s_ml = reinterpret_cast<float2*>(smem + C::kOffV);
  static_assert((14 + 2 * C::kKStages + 2 * C::kVStages + 2 * C::kSlots) * 8 + 4 <= 384, "the barriers' place");

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // (the shuffle: the same in all lanes, also to the compiler)
  constexpr int kUnpackWarp = C::kSoftmaxWarps, kIssueWarp = kUnpackWarp + 4, kCopyWarp = kIssueWarp + TILES;
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) mbar_init(&bar_q[t], 4);
    for (int i = 0; i < C::kKStages; ++i) {
      mbar_init(&bar_kfull[i], 4);
      mbar_init(&bar_kfree[i], TILES);
      mbar_init(&bar_vfull[i], 4);
      mbar_init(&bar_vfree[i], TILES);
    }
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&bar_raw[i], 1);
      mbar_init(&bar_used[i], 4);
    }
    for (int t = 0; t < 4; ++t) {
      mbar_init(&bar_s[t], 1);
      mbar_init(&bar_p[t], 4);
      mbar_init(&bar_o[t], 1);
    }
    fence_barrier_init();
  }
  if (warp == kIssueWarp) tmem_alloc<TILES * kTileCols>(s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // ---- this block's share ----
  const Share share = share_of<MODE>(p, blockIdx.x);
  int hk = share.item % static_cast<unsigned>(p.num_kv_heads);
  const unsigned of_rows = share.item / static_cast<unsigned>(p.num_kv_heads);
  int b = of_rows % static_cast<unsigned>(p.batch), rb = p.row_blocks - 1 - static_cast<int>(of_rows / static_cast<unsigned>(p.batch));  // the last rows see most keys: first
  asm volatile("" : "+r"(hk), "+r"(b), "+r"(rb));  // (as they are, not worked out again inside the loops: INT8 spilled, 1 to 2 % of a call)
  const int group = static_cast<unsigned>(p.num_heads) / static_cast<unsigned>(p.num_kv_heads);
  pdl_wait();
  // Only now: what is launched next may read what this kernel's predecessors wrote (the tail kernel does, ahead of its own wait)
  pdl_launch_dependents();

  Portion portion = p.shared_blocks > 0 ? Portion{0, p.num_tokens, 0} : portion_of(p.cu, p.lengths, b, p.num_tokens);
  portion.count = min(portion.count, p.max_seqlen);
  const int n_rows = portion.count * group;
  const int row_base = rb * (TILES * kRows);
  const bool any = row_base < n_rows;
  int n_keys;  // that the block's last row sees
  if (p.shared_blocks > 0) {
    n_keys = p.shared_blocks * kPage;
  } else {
    const int last = min(n_rows, row_base + TILES * kRows) - 1;
    n_keys = any ? min(max(portion.first + last / group + 1, 0), p.max_blocks * kPage) : 0;
  }
  const int n_pages = (n_keys + kPage - 1) / kPage;
  // (nsplit <= 128 splits of at most 2^24 pages: 32 bits hold the products)
  int page0 = static_cast<int>(share.split * n_pages / share.nsplit);
  int n_mine = any ? static_cast<int>((share.split + 1) * n_pages / share.nsplit) - page0 : 0;
  asm volatile("" : "+r"(page0), "+r"(n_mine));

  auto join_cluster = [&](int turn) {
    // The blocks of the cluster take turns over the rows, their softmax and unpacking warps too: lane = four dims
    cluster_sync();
    const int rows = min(n_rows - row_base, kRows);
#pragma unroll 1
    for (int i = static_cast<int>(share.split) + p.cluster * turn; i < rows; i += p.cluster * 8) {
      const float* at = reinterpret_cast<const float*>(smem + i * (kD * 4) + ((lane ^ (i & 7)) << 4));
      float4 x[kMostCluster];
      float2 ml[kMostCluster];
#pragma unroll
      for (int k = 0; k < kMostCluster; ++k) {
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        ml[k] = make_float2(-CUDART_INF_F, 0.f);
        if (k < p.cluster) {
          const uint2 w = peer_u2(s_ml + i, k);
          ml[k] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
          x[k] = peer_f32x4(at, k);
        }
      }
      float M = -CUDART_INF_F, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kMostCluster; ++k) M = fmaxf(M, ml[k].x);
      const float ref = M == -CUDART_INF_F ? 0.f : M;
#pragma unroll
      for (int k = 0; k < kMostCluster; ++k) {
        const float w = ml[k].y * ex2(ml[k].x - ref);
        L += w;
        acc.x = fmaf(x[k].x, w, acc.x); acc.y = fmaf(x[k].y, w, acc.y); acc.z = fmaf(x[k].z, w, acc.z); acc.w = fmaf(x[k].w, w, acc.w);
      }
      const int row = row_base + i, t = row / group, h = hk * group + row - t * group;
      const long long token = portion.start + t;
      reinterpret_cast<uint2*>(p.out + token * p.out_stride + static_cast<long long>(h) * kD)[lane] = scaled_h4(acc, L);
    }
    cluster_sync();  // no block leaves while another reads its rows
  };

  if (warp >= kUnpackWarp && warp < kIssueWarp) {
    // ===================================== unpacking =====================================
    if constexpr (C::kShares) set_max_regs<false, kUnpackRegs>();
    const int t = threadIdx.x - 32 * kUnpackWarp;
    // thread: key t / 2, dims 64 (t % 2) .. + 63.  The odd threads take their words in the other order, so that eight neighbours meet every bank once.
    const int key = t >> 1, part = t & 1;
    const uint32_t row_at = part * kKvHalf + key * 128, swizzle = key & 7;
    const long long* ptrs = p.kv_pointers + static_cast<long long>(b) * 2 * p.max_blocks + page0;
    asm volatile("" : "+l"(ptrs));  // (not worked out again for every page either)
    constexpr int kWords = BITS / 2;  // 16-byte words of a thread's 64 codes
    struct Raw {
      uint4 k[kWords], v[kWords];
      __half ks, kz, vs, vz;
    };
    // a page's codes, scales and zeros out of the pages ...
    const long long codes = G::codes_at(hk) + t * (G::kRow / 2), scale = G::scales_at(hk, p.num_kv_heads) + key * 2, zero = G::zeros_at(hk, p.num_kv_heads) + key * 2;
    long long kp = 0, vp = 0;  // lane i: page 32 n + i
    // INT8: K's codes follow as soon as the page's own are unpacked, while its values are; INT4, half as many, all behind both (30 tokens behind 30000, us: INT8 32.9
    // all behind both, 32.2 so; INT4 27.1 and 27.9)
    constexpr bool kEarly = !C::kRing && BITS == 8;
    const uint8_t *k_page = nullptr, *v_page = nullptr;
    auto turn = [&](Raw& r, int j) {  // to page j: its scales and zeros
      if (j >= n_mine) return;
      if ((j & 31) == 0 && j + lane < n_mine) {
        kp = __ldcg(ptrs + j + lane);
        vp = __ldcg(ptrs + p.max_blocks + j + lane);
      }
      k_page = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, kp, j & 31));
      v_page = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, vp, j & 31));
      r.ks = __ldcg(reinterpret_cast<const __half*>(k_page + scale));
      r.kz = __ldcg(reinterpret_cast<const __half*>(k_page + zero));
      r.vs = __ldcg(reinterpret_cast<const __half*>(v_page + scale));
      r.vz = __ldcg(reinterpret_cast<const __half*>(v_page + zero));
    };
    auto fetch = [&](uint4 (&code)[kWords], const uint8_t* page) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) code[i] = __ldcg(reinterpret_cast<const uint4*>(page + codes) + (i ^ (part * (kWords / 2))));
    };
    // ... or out of their raw slot
    constexpr int kSlots = C::kRing ? C::kSlots : 1;
    auto take = [&](Raw& r, int j) {
      const int slot = j % kSlots;
      const uint8_t* from = smem + C::kOffRaw + slot * C::kSlotBytes;
      mbar_wait(&bar_raw[slot], static_cast<uint32_t>(j / kSlots) & 1u);
      const __half* meta = reinterpret_cast<const __half*>(from + C::kMeta) + key;
      r.ks = meta[0]; r.kz = meta[64]; r.vs = meta[128]; r.vz = meta[192];
      const uint4* k = reinterpret_cast<const uint4*>(from + t * (G::kRow / 2));
      const uint4* v = reinterpret_cast<const uint4*>(from + C::kCodes + t * (G::kRow / 2));
#pragma unroll
      for (int i = 0; i < kWords; ++i) r.k[i] = k[i ^ (part * (kWords / 2))];
#pragma unroll
      for (int i = 0; i < kWords; ++i) r.v[i] = v[i ^ (part * (kWords / 2))];
    };
    auto unpack = [&](const uint4 (&raw)[kWords], __half2 s2, __half2 c2, __half2 low2, uint8_t* dst) {
      uint8_t* row = dst + row_at;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const int at = i ^ (part * (kWords / 2));
        const uint32_t words[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        auto put = [&](int chunk, const __half2 (&x)[4]) {
          *reinterpret_cast<uint4*>(row + ((chunk ^ swizzle) << 4)) = make_uint4(as_u32(x[0]), as_u32(x[1]), as_u32(x[2]), as_u32(x[3]));
        };
        if constexpr (BITS == 4) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            __half2 u[4];
            codes_of_word4(words[k], u);
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = __hfma2(u[e], s2, c2);
            put(4 * at + k, u);  // dims 0 4 1 5 2 6 3 7 of eight: the queries lie in the same order, O's columns come out in it
          }
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            __half2 lo[2], hi[2];
            codes_of_word8(words[2 * k], low2, lo);
            codes_of_word8(words[2 * k + 1], low2, hi);
            __half2 u[4] = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = __hfma2(u[e], s2, c2);
            put(2 * at + k, u);
          }
        }
      }
      fence_proxy_async();
      __syncwarp();
    };
    auto step = [&](Raw& raw, int j) {
      const bool live = (page0 + j) * kPage + key < n_keys;
      // (K, V)
      __half2 s = __halves2half2(raw.ks, raw.vs), c = __halves2half2(raw.kz, raw.vz), most;  // what the row's codes stand for is no further from 0
      if constexpr (BITS == 4) {
        c = __hmul2(__hneg2(s), c);
        most = __hmax2(__habs2(__hfma2(s, __float2half2_rn(15.f), c)), __habs2(c));
      } else {
        // (taken 2^-8 more: its three roundings are others than those of the numbers below, 2^-11 each)
        most = __hmul2(__hmul2(__habs2(s), __float2half2_rn(1.f + 1.f / 256.f)), __hmax2(__habs2(c), __habs2(__hsub2(__float2half2_rn(255.f), c))));
      }
      const uint32_t endless = as_u32(most) & 0x7c007c00u;
      const bool wide = live && ((endless & 0xffffu) == 0x7c00u || endless >= 0x7c000000u);
      if (!live) s = c = __float2half2_rn(0.f);
      if (__any_sync(0xffffffffu, wide)) {
        // A row of K or V whose scale or zero is no finite number stands for NaN: the key's score is NaN then (and goes where the key is masked), its value 0, so
        // that a weight of 0 in a row that does not see it stays 0.  Otherwise what counts is the codes that the row has (a row of one value is held as 1 x that
        // value, and 15 or 255 of it would be past fp16): one with a number past fp16's all the same (the rounded scale of a row that reaches the ends of fp16 does
        // that) is taken as much smaller as brings it inside, for an infinity times a weight of 0 would be NaN as well.  65520 is the least that rounds to infinity;
        // 65376 leaves room for the roundings of the smaller scale and zero (INT4: 15 x 4 + 16 at most; INT8: 2^-11 of each).
        const float2 sf = __half22float2(s), cf = __half22float2(c);
        auto inside = [&](const uint4 (&code)[kWords], float scale, float other) {
          uint32_t lo = 0xffffffffu, hi = 0u;
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            const uint32_t words[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (BITS == 4) {
                const uint32_t even = words[k] & 0x0f0f0f0fu, odd = (words[k] >> 4) & 0x0f0f0f0fu;
                lo = __vminu4(lo, __vminu4(even, odd));
                hi = __vmaxu4(hi, __vmaxu4(even, odd));
              } else {
                lo = __vminu4(lo, words[k]);
                hi = __vmaxu4(hi, words[k]);
              }
            }
          }
          lo = __vminu4(lo, __shfl_xor_sync(0xffffffffu, lo, 1));  // the row's other thread
          hi = __vmaxu4(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
#pragma unroll
          for (int m = 16; m >= 8; m >>= 1) {
            lo = __vminu4(lo, lo >> m | lo << (32 - m));
            hi = __vmaxu4(hi, hi >> m | hi << (32 - m));
          }
          const float least = static_cast<float>(lo & 255u), largest = static_cast<float>(hi & 255u);
          float end;
          if constexpr (BITS == 4) {
            end = fmaxf(fabsf(fmaf(scale, least, other)), fabsf(fmaf(scale, largest, other)));
          } else {  // with the rounding of what the zero leaves behind its whole part
            const float rest = fabsf(other - rintf(fminf(fmaxf(other, -1024.f), 1024.f)));
            end = fabsf(scale) * (fmaxf(fabsf(least - other), fabsf(largest - other)) + rest * 4.8828125e-4f);
          }
          return end >= 65520.f ? 65376.f / end : 1.f;
        };
        const float k = inside(raw.k, sf.x, cf.x), v = inside(raw.v, sf.y, cf.y);
        auto none = [](__half h) { return (__half_as_ushort(h) & 0x7c00u) == 0x7c00u; };
        if (wide) {
          if (none(__low2half(s)) || none(__high2half(s)) || none(__low2half(c)) || none(__high2half(c))) {
            s = c = __halves2half2(__ushort_as_half(0x7fffu), __ushort_as_half(0));
          } else {
            s = __floats2half2_rn(sf.x * k, sf.y * v);
            if constexpr (BITS == 4) c = __floats2half2_rn(cf.x * k, cf.y * v);
          }
        }
      }
      __half2 low = c;
      if constexpr (BITS == 8) {
        // s (u - z) in one rounding: u less the nearest whole number to z, exact, times s, plus s times the rest of z (at most 1 / 2; a zero further than 1024 from 0,
        // which is whole, leaves more there, and that product is rounded too).  u - z itself may have more bits than fp16: 255 less a zero of 54.6875 does
        const __half2 end = __float2half2_rn(1024.f), whole = h2rint(__hmax2(__hmin2(c, end), __hneg2(end)));
        low = __hneg2(__hadd2(whole, end));
        c = __hmul2(s, __hsub2(whole, c));
      }
      if constexpr (kEarly) turn(raw, j + 1);
      const int ks_at = j % C::kKStages, vs_at = j % C::kVStages;
      mbar_wait(&bar_kfree[ks_at], (static_cast<uint32_t>(j / C::kKStages) & 1u) ^ 1u);
      unpack(raw.k, __low2half2(s), __low2half2(c), __low2half2(low), smem + C::kOffK + ks_at * kKvBytes);
      if (lane == 0) mbar_arrive(&bar_kfull[ks_at]);
      if constexpr (kEarly) {
        if (j + 1 < n_mine) fetch(raw.k, k_page);
      }
      mbar_wait(&bar_vfree[vs_at], (static_cast<uint32_t>(j / C::kVStages) & 1u) ^ 1u);
      unpack(raw.v, __high2half2(s), __high2half2(c), __high2half2(low), smem + C::kOffV + vs_at * kKvBytes);
      if (lane == 0) mbar_arrive(&bar_vfull[vs_at]);
      if constexpr (kEarly) {
        if (j + 1 < n_mine) fetch(raw.v, v_page);
      }
    };
    Raw raw;
    if constexpr (C::kRing) {
      for (int j = 0; j < n_mine; ++j) {
        take(raw, j);
        step(raw, j);
        if (lane == 0) mbar_arrive(&bar_used[j % kSlots]);
      }
    } else {
      auto all = [&](int j) {
        if (j >= n_mine) return;
        turn(raw, j);
        fetch(raw.k, k_page);
        fetch(raw.v, v_page);
      };
      all(0);
      for (int j = 0; j < n_mine; ++j) {
        step(raw, j);
        if constexpr (!kEarly) all(j + 1);
      }
    }
    if constexpr (MODE == kCluster) join_cluster(4 + warp - kUnpackWarp);
  } else if (warp >= kIssueWarp) {
    if constexpr (C::kShares) set_max_regs<false, kIssueRegs>();
    if (C::kRing && warp == kCopyWarp) {
      // ===================================== copies: six of a page, a lane each =====================================
      constexpr int kSlots = C::kRing ? C::kSlots : 1;
      const long long* kptrs = p.kv_pointers + static_cast<long long>(b) * 2 * p.max_blocks + page0;
      const long long* vptrs = kptrs + p.max_blocks;
      long long kp = 0, vp = 0;  // lane i: page 32 n + i
      // codes, scales, zeros of K (even lanes) and of V
      const int what = lane >> 1, of_v = lane & 1;
      const long long from = what == 0 ? G::codes_at(hk) : what == 1 ? G::scales_at(hk, p.num_kv_heads) : G::zeros_at(hk, p.num_kv_heads);
      const int to = what == 0 ? of_v * C::kCodes : C::kMeta + of_v * 256 + (what - 1) * 128, bytes = what == 0 ? C::kCodes : 128;
      for (int j = 0; j < n_mine; ++j) {
        if ((j & 31) == 0 && j + lane < n_mine) {
          kp = __ldcg(kptrs + j + lane);
          vp = __ldcg(vptrs + j + lane);
        }
        const long long k = __shfl_sync(0xffffffffu, kp, j & 31), v = __shfl_sync(0xffffffffu, vp, j & 31);
        const int slot = j % kSlots;
        mbar_wait(&bar_used[slot], (static_cast<uint32_t>(j / kSlots) & 1u) ^ 1u);
        if (lane == 0) mbar_expect_tx(&bar_raw[slot], C::kSlotBytes);
        __syncwarp();
        if (lane < 6) bulk_copy_g2s(smem + C::kOffRaw + slot * C::kSlotBytes + to, reinterpret_cast<const uint8_t*>(of_v ? v : k) + from, bytes, &bar_raw[slot]);
      }
    } else if (warp < kIssueWarp + TILES && n_mine > 0) {
      // ===================================== products: a warp per tile, all its lanes in step and one of them issuing =====================================
      // (a lane that is alone in its branch takes 90 cycles for an instruction's descriptors, twelve of them a page and tile)
      constexpr uint32_t idesc_qk = idesc_f16(kRows, kPage, 0u), idesc_pv = idesc_f16(kRows, kD, 1u);
      const int t = warp - kIssueWarp;
      const bool leader = elect_one();
      const uint32_t base = smem_u32(smem), cols = tmem + t * kTileCols;
      const uint64_t q_desc = umma_desc_sw128(base + t * kQBytes), k_desc = umma_desc_sw128(base + C::kOffK), v_desc = desc_sw128_mn(base + C::kOffV, kKvHalf);
      auto scores = [&](int j) {
        const int st = j % C::kKStages;
        mbar_wait(&bar_kfull[st], static_cast<uint32_t>(j / C::kKStages) & 1u);
        // over the P of the page before the one before, once that has been taken
        if (j >= 2) mbar_wait(&bar_o[t * 2 + (j & 1)], static_cast<uint32_t>((j - 2) >> 1) & 1u);
        tc_fence_after();
        if (leader) {
          const uint64_t kd = k_desc + static_cast<uint64_t>(st * (kKvBytes >> 4));
          const uint32_t to = cols + (j & 1) * kPage;
#pragma unroll
          for (int ks = 0; ks < kD / 16; ++ks)
            mma_f16_ss(to, q_desc + ((ks >> 2) * (kQBytes / 2 >> 4) + (ks & 3) * 2), kd + ((ks >> 2) * (kKvHalf >> 4) + (ks & 3) * 2), idesc_qk, ks > 0 ? 1u : 0u);
          umma_commit(&bar_s[t * 2 + (j & 1)]);
          umma_commit(&bar_kfree[st]);
        }
        __syncwarp();
      };
      mbar_wait(&bar_q[t], 0);
      scores(0);
      if (n_mine > 1) scores(1);
      for (int j = 0; j < n_mine; ++j) {
        const int st = j % C::kVStages;
        mbar_wait(&bar_vfull[st], static_cast<uint32_t>(j / C::kVStages) & 1u);
        mbar_wait(&bar_p[t * 2 + (j & 1)], static_cast<uint32_t>(j >> 1) & 1u);
        tc_fence_after();
        if (leader) {
          const uint64_t vd = v_desc + static_cast<uint64_t>(st * (kKvBytes >> 4));
          const uint32_t from = cols + (j & 1) * kPage;
#pragma unroll
          for (int kk = 0; kk < kPage / 16; ++kk) mma_f16_ts(cols + kColO, from + kk * 8, vd + kk * (2048 >> 4), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&bar_o[t * 2 + (j & 1)]);
          umma_commit(&bar_vfree[st]);
        }
        __syncwarp();
        if (j + 2 < n_mine) scores(j + 2);
      }
    }
  } else {
    // ===================================== queries, softmax, results: thread = row =====================================
    if constexpr (C::kShares) set_max_regs<true, kSoftmaxRegs>();
    const int tile = warp >> 2, quarter = warp & 3;
    const int first_row = row_base + tile * kRows + quarter * 32;
    const bool alive = first_row < n_rows;  // warp-uniform; a warp without rows lets its part of Q, S and P be what it is
    const int r = first_row + lane, tok = r / group, head = hk * group + r - tok * group;
    const bool row_is = r < n_rows;
    if (alive && n_mine > 0) {  // (no page: the results' zeros would meet another warp's late queries in the same shared memory, for no product stands between them)
      // half a warp a row, 16 bytes a lane, all rows on their way together; where a row begins is worked out by the lane whose row it is
      uint8_t* dst = smem + tile * kQBytes;
      const int c = lane & 15;
      const unsigned long long mine = row_is ? reinterpret_cast<unsigned long long>(p.q + (portion.start + tok) * p.q_stride + static_cast<long long>(head) * kD) : 0ull;
      uint4 x[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const uint4* row = reinterpret_cast<const uint4*>(__shfl_sync(0xffffffffu, mine, 2 * k + (lane >> 4)));
        x[k] = row ? __ldcg(row + c) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int in_tile = quarter * 32 + 2 * k + (lane >> 4);
        if constexpr (BITS == 4)  // the order in which the keys' dims are unpacked
          x[k] = make_uint4(__byte_perm(x[k].x, x[k].z, 0x5410), __byte_perm(x[k].x, x[k].z, 0x7632), __byte_perm(x[k].y, x[k].w, 0x5410),
                            __byte_perm(x[k].y, x[k].w, 0x7632));
        *reinterpret_cast<uint4*>(dst + (c >> 3) * (kQBytes / 2) + in_tile * 128 + (((c & 7) ^ (in_tile & 7)) << 4)) = x[k];
      }
      fence_proxy_async();
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar_q[tile]);
    // the last position that the row sees, and the lowest of the warp's rows (one that is no row: its numbers go nowhere)
    int limit = n_keys - 1;
    if (row_is) limit = p.shared_blocks > 0 ? min(max(__ldcg(p.lengths + tok), 0), n_keys) - 1 : min(portion.first + tok, n_keys - 1);
    int lowest = limit;
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) lowest = min(lowest, __shfl_xor_sync(0xffffffffu, lowest, m));
    const uint32_t t_s = tmem + tile * kTileCols + (static_cast<uint32_t>(quarter * 32) << 16), t_o = t_s + kColO;
    float m_used = -CUDART_INF_F, l = 0.f;  // what O and the sum are expressed against (log2 units)
    for (int j = 0; j < n_mine; ++j) {
      const uint32_t s_at = t_s + (j & 1) * kPage;
      uint32_t x[2][32], w[32];
      mbar_wait(&bar_s[tile * 2 + (j & 1)], static_cast<uint32_t>(j >> 1) & 1u);
      tc_fence_after();
      if (alive) {
        tmem_ld_32x32b_x32(s_at, x[0]);
        tmem_ld_32x32b_x32(s_at + 32, x[1]);
        tmem_wait_ld();
        const int key0 = (page0 + j) * kPage;
        if (key0 + kPage - 1 > lowest) {  // warp-uniform
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (key0 + c * 32 + i > limit) x[c][i] = 0xff800000u;  // -inf
        }
        float top[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2) top[(i >> 1) & 3] = max3(top[(i >> 1) & 3], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
        const float m_page = fmaxf(max3(top[0], top[1], top[2]), top[3]) * p.scale_log2;
        if (j == 0) {
          m_used = m_page - kLift;
        } else {
          const bool grow = m_page - m_used > kLift + kRescale;  // also from -inf; a row that has seen nothing yet and sees nothing here: NaN, no
          if (__any_sync(0xffffffffu, grow)) {
            mbar_wait(&bar_o[tile * 2 + ((j - 1) & 1)], static_cast<uint32_t>((j - 1) >> 1) & 1u);  // the O += P V before
            tc_fence_after();
            const float m_new = grow ? m_page - kLift : m_used;
            const float alpha = grow ? ex2(m_used - m_new) : 1.f;
#pragma unroll 1
            for (int c = 0; c < kD / 32; ++c) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(t_o + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st_x32(t_o + c * 32, o);
            }
            l *= alpha;
            m_used = m_new;
          }
        }
        const float m_ref = m_used == -CUDART_INF_F ? 0.f : m_used;  // a row without any key so far: its weights are exp2(-inf) = 0
        const f2 scale2 = pack2(p.scale_log2, p.scale_log2), m2 = pack2(-m_ref, -m_ref);
        f2 sum[2] = {pack2(l, 0.f), pack2(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const float2 e = unpack2(fma2(pack2(__uint_as_float(x[i >> 5][i & 31]), __uint_as_float(x[i >> 5][(i & 31) + 1])), scale2, m2));
          const float p0 = ex2(e.x), p1 = ex2(e.y);
          sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pack2(p0, p1));
          w[i >> 1] = as_u32(__floats2half2_rn(p0, p1));
        }
        const float2 two = unpack2(add2(sum[0], sum[1]));
        l = two.x + two.y;
        tmem_st_x32(s_at, w);
        tmem_wait_st();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_p[tile * 2 + (j & 1)]);
    }
    if (alive) {
      if (n_mine > 0) mbar_wait(&bar_o[tile * 2 + ((n_mine - 1) & 1)], static_cast<uint32_t>((n_mine - 1) >> 1) & 1u);
      tc_fence_after();
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // a row without keys: zeros
      const long long token = portion.start + tok;
      // eight dims in turn of the row's 128
      auto eight = [&](const uint32_t (&o)[32], int e, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(o[e * 8 + (BITS == 4 ? (i < 4 ? 2 * i : 2 * i - 7) : i)]) * inv;
      };
      auto fetch = [&](uint32_t (&o)[32], int c) {
        if (n_mine > 0) {
          tmem_ld_32x32b_x32(t_o + c * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
      };
      // A partial row: where it goes, in rows of 128 numbers.  (The block's number is read again, so that the loop above holds nothing of it: it has no register to
      // spare)
      bool partial = false;
      long long at = 0;
      unsigned long long to = 0ull;
      if constexpr (MODE != kCluster) {
        if constexpr (MODE == kPartial) {
          unsigned block;
          asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(block));
          const Share mine = share_of<MODE>(p, block);
          partial = block >= static_cast<unsigned>(p.split_from);
          const int row = p.split_from == 0 ? static_cast<int>(token) * p.num_heads + head
                                            : static_cast<int>(mine.item - p.split_from) * (TILES * kRows) + (tile * kRows + quarter * 32 + lane);
          at = static_cast<long long>(row) * p.parts + mine.split;
        }
        if (row_is) to = partial ? reinterpret_cast<unsigned long long>(p.part + at * kD)
                                 : reinterpret_cast<unsigned long long>(p.out + token * p.out_stride + static_cast<long long>(head) * kD);
      }
      if constexpr (MODE != kWhole && TILES == 1) {
        // fp32 rows of 512 bytes over Q and K, all of whose products have retired
        static_assert(kRows * kD * 4 <= C::kOffV, "rows' maxima and sums lie behind the rows");
        uint8_t* const rows = smem + quarter * 32 * (kD * 4);
        auto chunk = [&](int row, int i) { return reinterpret_cast<float4*>(rows + row * (kD * 4) + ((i ^ (row & 7)) << 4)); };
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          fetch(o, c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float f[8];
            eight(o, e, f);
            *chunk(lane, c * 8 + 2 * e) = make_float4(f[0], f[1], f[2], f[3]);
            *chunk(lane, c * 8 + 2 * e + 1) = make_float4(f[4], f[5], f[6], f[7]);
          }
        }
        if constexpr (MODE == kCluster) {
          s_ml[quarter * 32 + lane] = make_float2(m_used, l);
        } else {  // a warp a row
          __syncwarp();
          const int many = min(32, n_rows - first_row);
#pragma unroll 8
          for (int k = 0; k < many; ++k) {
            const unsigned long long row = __shfl_sync(0xffffffffu, to, k);
            const float4 x = *chunk(k, lane);
            if (partial) reinterpret_cast<float4*>(row)[lane] = x;
            else reinterpret_cast<uint2*>(row)[lane] = make_uint2(results(x.x, x.y), results(x.z, x.w));
          }
        }
      } else {
        // Through shared memory (the tile's queries are done with), so that half a warp stores a whole row, or half a row of fp32
        uint8_t* mine = smem + tile * kQBytes + quarter * (kQBytes / 4);
        auto put = [&](int chunk, uint4 x) { *reinterpret_cast<uint4*>(mine + lane * 256 + ((chunk ^ (lane & 7)) << 4)) = x; };
        auto store = [&](int behind) {
          __syncwarp();
#pragma unroll 4
          for (int k = 0; k < 32; k += 2) {
            const int in = k + (lane >> 4), chunk = lane & 15;
            uint4* row = reinterpret_cast<uint4*>(__shfl_sync(0xffffffffu, to, in));
            const uint4 v = *reinterpret_cast<const uint4*>(mine + in * 256 + ((chunk ^ (in & 7)) << 4));
            if (row) row[behind + chunk] = v;
          }
          __syncwarp();
        };
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          fetch(o, c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float f[8];
            eight(o, e, f);
            if (MODE == kPartial && partial) {
              put((c & 1) * 8 + 2 * e, make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])));
              put((c & 1) * 8 + 2 * e + 1, make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7])));
            } else {
              put(c * 4 + e, make_uint4(results(f[0], f[1]), results(f[2], f[3]), results(f[4], f[5]), results(f[6], f[7])));
            }
          }
          if (MODE == kPartial && partial && c == 1) store(0);
        }
        store(MODE == kPartial && partial ? 16 : 0);
      }
      if (partial && row_is) p.part_ml[at] = make_float2(m_used, l);
    }
    if constexpr (MODE == kCluster) join_cluster(warp);
  }
  if constexpr (MODE == kCluster) {
    if (warp >= kIssueWarp) {  // the other warps' two waits
      cluster_sync();
      cluster_sync();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kIssueWarp) tmem_dealloc<TILES * kTileCols>(tmem);
}

// ------------------------------------------------------------------------------------------------------------------------
// partial rows of a split joined: a warp, lane = 4 dims.  Returns the sum and the maximum that acc is expressed against.
// ------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void join_rows(const float* part, const float2* ml, int nsplit, float& M, float& L, float4& acc) {
  const int lane = threadIdx.x & 31;
  for (int s0 = 0; s0 < nsplit; s0 += 32) {
    const int n = min(32, nsplit - s0);
    const float4* rows = reinterpret_cast<const float4*>(part + static_cast<long long>(s0) * kD) + lane;
    float4 x[8];
    auto fetch = [&](int s) {
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = s + k < n ? __ldcg(rows + (s + k) * (kD / 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    fetch(0);  // on their way together with the maxima and sums
    const float2 mine = lane < n ? __ldcg(ml + s0 + lane) : make_float2(-CUDART_INF_F, 0.f);
    float m = mine.x;
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    const float m_new = fmaxf(M, m), ref = m_new == -CUDART_INF_F ? 0.f : m_new;
    const float old = ex2(M - ref), weight = mine.y * ex2(mine.x - ref);  // of O / sum
    float sum = weight;
#pragma unroll
    for (int k = 16; k >= 1; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    L = fmaf(L, old, sum);
    acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
    M = m_new;
    for (int s = 0; s < n; s += 8) {
      if (s > 0) fetch(s);
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // (behind the last split: zeros with a weight of zero)
        const float ws = __shfl_sync(0xffffffffu, weight, (s + k) & 31);
        acc.x = fmaf(x[k].x, ws, acc.x); acc.y = fmaf(x[k].y, ws, acc.y); acc.z = fmaf(x[k].z, ws, acc.z); acc.w = fmaf(x[k].w, ws, acc.w);
      }
    }
  }
}

// The rows that were split (all of them, by token and head; or those of some items), WARPS warps each (they take turns over the splits).  Rows behind the last
// sequence are left as they are.
template <int WARPS>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ TileParams p) {
  __shared__ __align__(16) float s_acc[4][kD];
  __shared__ float2 s_ml[4];
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned row = blockIdx.x * (4 / WARPS) + warp / WARPS;
  bool mine;
  long long token;
  int head;
  if (p.split_from == 0) {
    const unsigned t = row / static_cast<unsigned>(p.num_heads);
    token = t;
    head = static_cast<int>(row - t * p.num_heads);
    pdl_wait();
    const int b = t < static_cast<unsigned>(p.num_tokens) ? sequence_of(p.cu, p.batch, static_cast<int>(t)) : -1;
    mine = b >= 0 && static_cast<int>(t) - (p.cu ? p.cu[b] : b) < p.max_seqlen;
  } else {
    const unsigned behind = row / static_cast<unsigned>(p.block_rows), item = p.split_from + behind, of_rows = item / static_cast<unsigned>(p.num_kv_heads);
    const int hk = item - of_rows * p.num_kv_heads, b = of_rows % static_cast<unsigned>(p.batch), rb = p.row_blocks - 1 - static_cast<int>(of_rows / static_cast<unsigned>(p.batch));
    const int r = rb * p.block_rows + static_cast<int>(row - behind * p.block_rows), group = p.num_heads / p.num_kv_heads, tok = r / group;
    pdl_wait();
    const Portion portion = portion_of(p.cu, p.lengths, b, p.num_tokens);
    mine = tok < min(portion.count, p.max_seqlen);
    token = portion.start + tok;
    head = hk * group + r - tok * group;
  }
  float M = -CUDART_INF_F, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  // this warp's run of the splits
  const int part = warp % WARPS, s0 = p.parts * part / WARPS, s1 = p.parts * (part + 1) / WARPS;
  const long long at = static_cast<long long>(row) * p.parts + s0;
  if (mine) join_rows(p.part + at * kD, p.part_ml + at, s1 - s0, M, L, acc);
  if constexpr (WARPS > 1) {
    reinterpret_cast<float4*>(s_acc[warp])[lane] = acc;
    if (lane == 0) s_ml[warp] = make_float2(M, L);
    __syncthreads();
    if (!mine || part != 0) return;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) {
      const float2 ml = s_ml[warp + w];
      const float4 x = reinterpret_cast<const float4*>(s_acc[warp + w])[lane];
      const float m_new = fmaxf(M, ml.x), ref = m_new == -CUDART_INF_F ? 0.f : m_new, old = ex2(M - ref), wt = ex2(ml.x - ref);
      L = L * old + ml.y * wt;
      acc.x = fmaf(x.x, wt, acc.x * old); acc.y = fmaf(x.y, wt, acc.y * old); acc.z = fmaf(x.z, wt, acc.z * old); acc.w = fmaf(x.w, wt, acc.w * old);
      M = m_new;
    }
  }
  if (mine) reinterpret_cast<uint2*>(p.out + token * p.out_stride + static_cast<long long>(head) * kD)[lane] = scaled_h4(acc, L);
}

// ------------------------------------------------------------------------------------------------------------------------
// tail kernel: the pages behind the shared ones
//
// A warp takes half pages (32 keys) in turn.  Codes go into the products as they lie: a nibble or byte in the low bits of an fp16 word
// is the subnormal number u 2^-24, exact as an operand, so there is no conversion and nothing to take off again; scales, zeros and 2^24 are applied to scores and
// weights in fp32:  q.k = s 2^24 (q.u 2^-24) + c sum(q),  sum p v = 2^24 sum (p s) u 2^-24 + sum (p s) (c / s).
// ------------------------------------------------------------------------------------------------------------------------
constexpr int kTailWarps = 4, kMaxG = 8, kSlice = 32, kMaxCluster = 8;
constexpr int kOPitch = kD + 4;

// DEEP: more slices of a warp on their way, for calls of two blocks per multiprocessor at most; otherwise as many blocks as registers allow
template <int BITS, bool DEEP>
struct SliceCfg {
  static constexpr int kRow = Geom<BITS>::kRow;
  static constexpr int kCodes = kSlice * kRow;
  static constexpr int kOffV = kCodes, kOffMeta = 2 * kCodes;  // K scales, K zeros, V scales, V zeros: 64 bytes each
  static constexpr int kBytes = 2 * kCodes + 256;
  static constexpr int kSlots = !DEEP ? 2 : BITS == 4 ? 4 : 3;
  static constexpr int kWarpBytes = kSlots * kBytes;
  static_assert(kWarpBytes >= kMaxG * kOPitch * 4, "a warp's ring holds its partial rows at the end");
  static constexpr int kSmem = kTailWarps * kWarpBytes;
  // where 16-byte word c of a key's row lies: reads of K (rows p and p + 4) and transposing reads of V (one word of eight rows) meet every bank once
  static __device__ __forceinline__ uint32_t place(int row, int c) {
    if constexpr (BITS == 4) return (row >> 1) * 128 + (((row ^ (row >> 2)) & 1) * 4 + (c ^ ((row >> 1) & 3))) * 16;
    else return row * 128 + (c ^ (((row >> 2) & 1) | ((row & 3) << 1))) * 16;
  }
};

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t smem) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}
struct TailParams {
  const __half* q;
  __half* out;
  long long q_stride, out_stride;
  const long long* kv_pointers;
  const int* lengths;
  int batch, max_blocks, num_heads, num_kv_heads, shared_blocks, nsplit, cluster;
  int common;  // pages from the first on that the first sequence's row names for all (0 where the tile kernel has read them: shared_blocks > 0)
  float scale_log2;
  const float* part;
  const float2* part_ml;
};

// SHARED: a block (and its cluster) per sequence and run of heads, the warps take turns over the slices; otherwise a warp for each of them, which saves the joining of
// warps where there are enough to fill the device.
template <int BITS, bool SHARED, bool DEEP>
__global__ void __launch_bounds__(32 * kTailWarps, DEEP ? 2 : BITS == 4 ? 4 : 3) tail_kernel(const __grid_constant__ TailParams p) {
  static_assert(SHARED || !DEEP, "a warp for each run of heads goes with many of them");
  using SC = SliceCfg<BITS, DEEP>;
  using G = Geom<BITS>;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(16) __half s_queries[(SHARED ? 1 : kTailWarps) * kMaxG * kD];
  __shared__ float s_m[kTailWarps][kMaxG], s_l[kTailWarps][kMaxG];
  __shared__ float2 s_meta[kTailWarps][2][kSlice];
  __shared__ __align__(16) float s_o[SHARED ? kMaxG * kD : 4];  // the block's rows
  __shared__ float s_bm[kMaxG], s_bl[kMaxG];
  const int group = p.num_heads / p.num_kv_heads, parts = (group + kMaxG - 1) / kMaxG;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int rank = SHARED ? static_cast<int>(blockIdx.x) : 0;
  const int run = SHARED ? static_cast<int>(blockIdx.y) : static_cast<int>(blockIdx.x) * kTailWarps + warp;  // not SHARED: of all sequences
  const int runs = p.num_kv_heads * parts;
  const int b = SHARED ? static_cast<int>(blockIdx.z) : min(run / runs, p.batch - 1), of_b = SHARED ? run : run % runs;
  const bool live = SHARED || run < runs * p.batch;  // a warp past the last one walks an empty sequence
  const int hk = of_b / parts, part = of_b - hk * parts;
  const int h0 = hk * group + part * kMaxG, heads = live ? min(kMaxG, group - part * kMaxG) : 0;
  pdl_launch_dependents();
  // The tile kernel before this one started this one after its own wait: everything ahead of the tile kernel is there.  Without one, this kernel waits itself.
  if (p.nsplit == 0) pdl_wait();

  const int len = live ? min(max(__ldcg(p.lengths + b), 0), p.max_blocks * kPage) : 0;  // (whatever the table says: no difference below wraps)
  const int slices = max((len - p.shared_blocks * kPage + kSlice - 1) / kSlice, 0);
  // the cluster's blocks and their warps take turns over the slices
  const int stride = SHARED ? p.cluster * kTailWarps : 1, mine = SHARED ? rank * kTailWarps + warp : 0;
  const int n_my = slices > mine ? (slices - mine + stride - 1) / stride : 0;
  const long long* kptrs = p.kv_pointers + static_cast<long long>(b) * 2 * p.max_blocks + p.shared_blocks;
  uint8_t* ring = smem + warp * SC::kWarpBytes;
  const uint32_t ring_at = smem_u32(ring);
  const uint32_t lane_at = SC::place(lane * 16 / SC::kRow, lane * 16 % SC::kRow / 16);
  long long kp_l = 0, vp_l = 0;  // lane i: the pages of slices 32 n + i
  auto issue = [&](int u) {
    if ((u & 31) == 0 && u + lane < n_my) {
      const int page = (mine + (u + lane) * stride) >> 1;
      const long long* row = page < p.common ? p.kv_pointers : kptrs;
      kp_l = __ldcg(row + page);
      vp_l = __ldcg(row + p.max_blocks + page);
    }
    const int half = (mine + u * stride) & 1;
    const uint8_t* kp = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, kp_l, u & 31));
    const uint8_t* vp = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, vp_l, u & 31));
    const uint32_t dst = ring_at + (u % SC::kSlots) * SC::kBytes;
    const long long codes = G::codes_at(hk) + half * SC::kCodes + lane * 16;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < SC::kCodes / 512; ++i)
        cp_async16(dst + w * SC::kOffV + i * 512 + (BITS == 8 && (i & 1) ? lane_at ^ 16u : lane_at), (w ? vp : kp) + codes + i * 512);
    if (lane < 16) {
      const uint8_t* page_at = lane < 8 ? kp : vp;
      const long long meta = (lane & 4) ? G::zeros_at(hk, p.num_kv_heads) : G::scales_at(hk, p.num_kv_heads);
      cp_async16(dst + SC::kOffMeta + lane * 16, page_at + meta + half * 64 + (lane & 3) * 16);
    }
  };
#pragma unroll
  for (int u = 0; u < SC::kSlots; ++u) {
    if (u < n_my) issue(u);
    cp_async_commit();
  }
  // ---- the queries: 16 lanes a row ----
  __half* s_q = s_queries + (SHARED ? 0 : warp * kMaxG * kD);
  for (int i = SHARED ? static_cast<int>(threadIdx.x) : lane; i < kMaxG * 16; i += SHARED ? 32 * kTailWarps : 32) {
    const int r = i >> 4;
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (r < heads) x = __ldcg(reinterpret_cast<const uint4*>(p.q + b * p.q_stride + static_cast<long long>(h0 + r) * kD) + (i & 15));
    reinterpret_cast<uint4*>(s_q)[i] = x;
  }
  if constexpr (SHARED) __syncthreads();
  else __syncwarp();
  // Q as the B operand (n = head g) in the order of the codes: INT4 word w of a lane's 32 dims has nibbles (0, 4 | 1, 5), (2, 6 | 3, 7); INT8 (0, 1 | 2, 3)
  uint32_t qb0[8], qb1[8];
  float sumq0, sumq1;
  {
    uint32_t qw[16];
    const uint4* qv = reinterpret_cast<const uint4*>(s_q + g * kD + 32 * q4);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint4 t = qv[k];
      qw[4 * k] = t.x; qw[4 * k + 1] = t.y; qw[4 * k + 2] = t.z; qw[4 * k + 3] = t.w;
    }
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float2 f = __half22float2(as_h2(qw[k]));
      sum += f.x + f.y;
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    sumq0 = __shfl_sync(0xffffffffu, sum, 8 * q4);
    sumq1 = __shfl_sync(0xffffffffu, sum, 8 * q4 + 4);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      if constexpr (BITS == 4) {
        const int k0 = 4 * (s >> 1) + (s & 1);
        qb0[s] = __byte_perm(qw[k0], qw[k0 + 2], 0x5410);
        qb1[s] = __byte_perm(qw[k0], qw[k0 + 2], 0x7632);
      } else {
        qb0[s] = qw[2 * s];
        qb1[s] = qw[2 * s + 1];
      }
    }
  }
  constexpr float kUp = 16777216.f;  // 2^24
  float o[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, ref0 = -CUDART_INF_F, ref1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f, c0 = 0.f, c1 = 0.f;
  float s_top = 5.9604645e-8f;  // 2^-24, the smallest scale
  const int tokA = (g & 1) * 4 + (g >> 1);
  const uint32_t k_at = SC::place(tokA, BITS == 4 ? q4 : 2 * q4);
  const uint32_t v_at = SC::place((lane & 1) * 4 + ((lane >> 1) & 3) + (lane & 8), lane >> 4) + SC::kOffV;
  for (int u = 0; u < n_my; ++u) {
    cp_async_wait<SC::kSlots - 1>();
    __syncwarp();
    const uint32_t slot = (u % SC::kSlots) * SC::kBytes;
    const uint8_t* st = ring + slot;
    const int t0 = p.shared_blocks * kPage + (mine + u * stride) * kSlice;
    // Per key in fp32: (scale, c) for the scores, with the softmax scale; (scale, c / scale) for the values, whose c goes with the rounded weight as their codes do, so
    // that a weight's rounding is one of the value and not of its codes.  One that is no finite number makes both NaN.  Keys past the end: zeros
    {
      const __half* mp = reinterpret_cast<const __half*>(st + SC::kOffMeta) + lane;
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const __half s = mp[64 * w], z = mp[64 * w + 32];
        float2 f = make_float2(__half2float(s), -__half2float(z));
        if constexpr (BITS == 4) {
          f.y = __half2float(__hmul(__hneg(s), z));
          if (w == 1) f.y = __fdividef(f.y, f.x == 0.f ? 1.f : f.x);
        } else if (w == 0) {
          f.y *= f.x;
        }
        const float none = fmaf(f.x, 0.f, f.y * 0.f);
        if (w == 0) f = make_float2(fmaf(f.x, p.scale_log2 * kUp, none), f.y * p.scale_log2);
        else f.y += none;
        if (t0 + lane >= len) f = make_float2(0.f, 0.f);
        s_meta[warp][w][lane] = f;
      }
    }
    __syncwarp();
    float sc[2][4] = {};
    float vmax = 0.f;  // of the values' scales
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint8_t* krow = st + c * 16 * SC::kRow + k_at;
      if constexpr (BITS == 4) {
        const uint4 ka = *reinterpret_cast<const uint4*>(krow), kb = *reinterpret_cast<const uint4*>(krow + 8 * SC::kRow);
        const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
        float high[4] = {};  // of the high nibbles, which are 16 u: by themselves, for q / 16 may not be an fp16 number
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t xa = wa[w], xb = wb[w], ta = xa >> 8, tb = xb >> 8;
          mma_16816(sc[c], xa & 0x000f000fu, xb & 0x000f000fu, ta & 0x000f000fu, tb & 0x000f000fu, qb0[2 * w], qb0[2 * w + 1]);
          mma_16816(high, xa & 0x00f000f0u, xb & 0x00f000f0u, ta & 0x00f000f0u, tb & 0x00f000f0u, qb1[2 * w], qb1[2 * w + 1]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[c][e] = fmaf(high[e], 0.0625f, sc[c][e]);
      } else {
        const uint8_t* krow1 = st + c * 16 * SC::kRow + (k_at ^ 16u);
        const uint4 ka0 = *reinterpret_cast<const uint4*>(krow), ka1 = *reinterpret_cast<const uint4*>(krow1);
        const uint4 kb0 = *reinterpret_cast<const uint4*>(krow + 8 * SC::kRow), kb1 = *reinterpret_cast<const uint4*>(krow1 + 8 * SC::kRow);
        const uint32_t wa[8] = {ka0.x, ka0.y, ka0.z, ka0.w, ka1.x, ka1.y, ka1.z, ka1.w};
        const uint32_t wb[8] = {kb0.x, kb0.y, kb0.z, kb0.w, kb1.x, kb1.y, kb1.z, kb1.w};
#pragma unroll
        for (int w = 0; w < 8; ++w)
          mma_16816(sc[c], __byte_perm(wa[w], 0u, 0x4140), __byte_perm(wb[w], 0u, 0x4140), __byte_perm(wa[w], 0u, 0x4342), __byte_perm(wb[w], 0u, 0x4342),
                    qb0[w], qb1[w]);
      }
    }
    float tl[2][4], vs[2][2], vc[2][2];
    const bool partial = t0 + kSlice > len;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float2 kA = s_meta[warp][0][c * 16 + tokA], kB = s_meta[warp][0][c * 16 + 8 + tokA];
      const float2 vA = s_meta[warp][1][c * 16 + tokA], vB = s_meta[warp][1][c * 16 + 8 + tokA];
      vs[c][0] = vA.x; vs[c][1] = vB.x; vc[c][0] = vA.y; vc[c][1] = vB.y;
      vmax = fmaxf(vmax, fmaxf(fabsf(vA.x), fabsf(vB.x)));
      tl[c][0] = fmaf(kA.x, sc[c][0], kA.y * sumq0);
      tl[c][1] = fmaf(kA.x, sc[c][1], kA.y * sumq1);
      tl[c][2] = fmaf(kB.x, sc[c][2], kB.y * sumq0);
      tl[c][3] = fmaf(kB.x, sc[c][3], kB.y * sumq1);
      if (partial) {
        if (t0 + c * 16 + tokA >= len) tl[c][0] = tl[c][1] = -CUDART_INF_F;
        if (t0 + c * 16 + 8 + tokA >= len) tl[c][2] = tl[c][3] = -CUDART_INF_F;
      }
    }
    // The weights are 2^up times those against the maximum, 2^up times the largest scale of a value so far 2^15: p s stays in the range of fp16 whatever the scales
    // are, and is no subnormal number where they are small.  (A slice always has a key, so the maxima are numbers.)
    float mh0 = fmaxf(fmaxf(tl[0][0], tl[0][2]), fmaxf(tl[1][0], tl[1][2])), mh1 = fmaxf(fmaxf(tl[0][1], tl[0][3]), fmaxf(tl[1][1], tl[1][3]));
    if (__any_sync(0xffffffffu, mh0 > m0 || mh1 > m1 || vmax > s_top)) {
#pragma unroll
      for (int m = 4; m <= 16; m <<= 1) {
        mh0 = fmaxf(mh0, __shfl_xor_sync(0xffffffffu, mh0, m));
        mh1 = fmaxf(mh1, __shfl_xor_sync(0xffffffffu, mh1, m));
        vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, m));
      }
      if (vmax > s_top) s_top = __uint_as_float((__float_as_uint(vmax) + 0x7fffffu) & 0x7f800000u);  // the next power of two
      const float up = static_cast<float>(142 - static_cast<int>(__float_as_uint(s_top) >> 23));
      m0 = fmaxf(m0, mh0);
      m1 = fmaxf(m1, mh1);
      const float a0 = ex2(ref0 - (m0 - up)), a1 = ex2(ref1 - (m1 - up));  // (nothing so far: 2^-inf)
      ref0 = m0 - up;
      ref1 = m1 - up;
      l0 *= a0; c0 *= a0; l1 *= a1; c1 *= a1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        o[i][0] *= a0; o[i][2] *= a0;
        o[i][1] *= a1; o[i][3] *= a1;
      }
    }
    uint32_t bp[2][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float pA0 = ex2(tl[c][0] - ref0), pA1 = ex2(tl[c][1] - ref1), pB0 = ex2(tl[c][2] - ref0), pB1 = ex2(tl[c][3] - ref1);
      l0 += pA0 + pB0; l1 += pA1 + pB1;
      // the products' operand: p s rounded to fp16
      const __half2 a = __floats2half2_rn(pA0 * vs[c][0], pA1 * vs[c][0]), b = __floats2half2_rn(pB0 * vs[c][1], pB1 * vs[c][1]);
      bp[c][0] = movmatrix_trans(as_u32(a));
      bp[c][1] = movmatrix_trans(as_u32(b));
      const float2 af = __half22float2(a), bf = __half22float2(b);
      c0 = fmaf(af.x, vc[c][0], fmaf(bf.x, vc[c][1], c0));
      c1 = fmaf(af.y, vc[c][0], fmaf(bf.y, vc[c][1], c1));
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int h = 0; h < kD / (256 / BITS); ++h) {
        uint32_t w[4];
        ldmatrix_x4_trans(w, ring_at + slot + c * 16 * SC::kRow + (v_at ^ (h * 32u)));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t lo = w[2 * e], hi = w[2 * e + 1];
          if constexpr (BITS == 4) {
            const int i = 4 * h + 2 * e;
            mma_16816(o[i], lo & 0x000f000fu, lo & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u, bp[c][0], bp[c][1]);
            const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
            mma_16816(o[i + 1], lo8 & 0x000f000fu, lo8 & 0x00f000f0u, hi8 & 0x000f000fu, hi8 & 0x00f000f0u, bp[c][0], bp[c][1]);
          } else {
            const int i = 2 * h + e;
            mma_16816(o[i], __byte_perm(lo, 0u, 0x4240), __byte_perm(lo, 0u, 0x4341), __byte_perm(hi, 0u, 0x4240), __byte_perm(hi, 0u, 0x4341), bp[c][0],
                      bp[c][1]);
          }
        }
      }
    }
    __syncwarp();
    if (u + SC::kSlots < n_my) issue(u + SC::kSlots);
    cp_async_commit();
  }
  // ---- a warp's partial rows into its ring: [head][place of the dim] ----
#pragma unroll
  for (int m = 4; m <= 16; m <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, m);
    l1 += __shfl_xor_sync(0xffffffffu, l1, m);
    c0 += __shfl_xor_sync(0xffffffffu, c0, m);
    c1 += __shfl_xor_sync(0xffffffffu, c1, m);
  }
  if (g == 0) {
    s_m[warp][2 * q4] = ref0; s_m[warp][2 * q4 + 1] = ref1;
    s_l[warp][2 * q4] = l0; s_l[warp][2 * q4 + 1] = l1;
  }
  {
    __syncwarp();
    float* so0 = reinterpret_cast<float*>(ring) + (2 * q4) * kOPitch + g;
    float* so1 = so0 + kOPitch;
    constexpr float kOdd = BITS == 4 ? kUp * 0.0625f : kUp;  // INT4: odd dims are the high nibbles, 16 u
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      so0[16 * i] = fmaf(o[i][0], kUp, c0); so0[16 * i + 8] = fmaf(o[i][2], kOdd, c0);
      so1[16 * i] = fmaf(o[i][1], kUp, c1); so1[16 * i + 8] = fmaf(o[i][3], kOdd, c1);
    }
  }
  if constexpr (!SHARED) {
    __syncwarp();
    if (p.nsplit > 0) pdl_wait();  // the prefix's partial rows
    for (int r = 0; r < heads; ++r) {
      const float* row = reinterpret_cast<const float*>(ring) + r * kOPitch;
      float x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // dim 4 lane + k
        const int d = 4 * lane + k;
        x[k] = row[BITS == 4 ? (d & ~31) | ((d >> 1 & 1) << 4) | ((d & 1) << 3) | ((d >> 2) & 7) : (d & ~15) | ((d & 1) << 3) | ((d >> 1) & 7)];
      }
      float M = s_m[warp][r], L = s_l[warp][r];
      float4 acc = make_float4(x[0], x[1], x[2], x[3]);
      const long long at = static_cast<long long>(b) * p.num_heads + h0 + r;
      if (p.nsplit > 0) join_rows(p.part + at * p.nsplit * kD, p.part_ml + at * p.nsplit, p.nsplit, M, L, acc);
      reinterpret_cast<uint2*>(p.out + b * p.out_stride + static_cast<long long>(h0 + r) * kD)[lane] = scaled_h4(acc, L);
    }
    return;
  }
  __syncthreads();
  // ---- the block's rows ----
  {
    // the dim whose partial sums lie at this thread's place
    const int t = threadIdx.x, d = BITS == 4 ? 32 * (t >> 5) + 4 * (t & 7) + 2 * ((t >> 4) & 1) + ((t >> 3) & 1) : 16 * (t >> 4) + 2 * (t & 7) + ((t >> 3) & 1);
    for (int r = 0; r < heads; ++r) {
      float M = -CUDART_INF_F;
#pragma unroll
      for (int w = 0; w < kTailWarps; ++w) M = fmaxf(M, s_m[w][r]);
      const float ref = M == -CUDART_INF_F ? 0.f : M;
      float acc = 0.f, L = 0.f;
#pragma unroll
      for (int w = 0; w < kTailWarps; ++w) {
        const float e = ex2(s_m[w][r] - ref);
        acc = fmaf(reinterpret_cast<const float*>(smem + w * SC::kWarpBytes)[r * kOPitch + t], e, acc);
        L = fmaf(s_l[w][r], e, L);
      }
      s_o[r * kD + d] = acc;
      if (t == 0) {
        s_bm[r] = M;
        s_bl[r] = L;
      }
    }
  }
  if (p.cluster > 1) cluster_sync();
  else __syncthreads();
  if (p.nsplit > 0) pdl_wait();  // the prefix's partial rows
  // ---- the cluster's blocks take turns over the heads, a block's warps too ----
  for (int r = rank + p.cluster * warp; r < heads; r += p.cluster * kTailWarps) {
    float M = -CUDART_INF_F, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < p.cluster; ++k) {
      const float m = p.cluster > 1 ? peer_f32(s_bm + r, k) : s_bm[r], sum = p.cluster > 1 ? peer_f32(s_bl + r, k) : s_bl[r];
      const float4 x = p.cluster > 1 ? peer_f32x4(s_o + r * kD + 4 * lane, k) : *reinterpret_cast<const float4*>(s_o + r * kD + 4 * lane);
      const float m_new = fmaxf(M, m), ref = m_new == -CUDART_INF_F ? 0.f : m_new;
      const float old = ex2(M - ref), w = ex2(m - ref);
      L = L * old + sum * w;
      acc.x = fmaf(x.x, w, acc.x * old); acc.y = fmaf(x.y, w, acc.y * old); acc.z = fmaf(x.z, w, acc.z * old); acc.w = fmaf(x.w, w, acc.w * old);
      M = m_new;
    }
    const long long row = static_cast<long long>(b) * p.num_heads + h0 + r;
    if (p.nsplit > 0) join_rows(p.part + row * p.nsplit * kD, p.part_ml + row * p.nsplit, p.nsplit, M, L, acc);
    reinterpret_cast<uint2*>(p.out + b * p.out_stride + static_cast<long long>(h0 + r) * kD)[lane] = scaled_h4(acc, L);
  }
  if (p.cluster > 1) cluster_sync();  // no block leaves while another reads its rows
}

// ------------------------------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------------------------------
template <auto Kern, typename Enough>
int allow_smem(int bytes, const char* what, Enough enough) {
  static bool done[kMaxDevices] = {};  // of this kernel
  bool& d = done[device_ordinal()];
  if (d) return QS_OK;
  cudaFuncAttributes attr{};
  const int ra = check_cuda(cudaFuncGetAttributes(&attr, Kern), what);
  if (ra) return ra;
  QS_REQUIRE(enough(attr.numRegs), "%s: %d registers per thread are fewer than the warpgroups share out", what, attr.numRegs);
  const int rc = check_cuda(cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
  if (rc == QS_OK) d = true;
  return rc;
}

// How a call over `rows` rows per kv head and sequence (`num_rows` of a kv head in all) and at most `pages` pages is cut: tiles per block, and splits of the pages.
// The cut whose time is estimated lowest: rounds of blocks over the device, each its pages and what comes ahead of the first and behind the last, and the joining of
// the splits: by a cluster of up to eight blocks (one tile of a prompt), by join_kernel, or in the tail kernel.  All items are split where they leave room in one
// round; in a prompt of more rounds the items of the last round, or of the last two, where those would not fill the device.  The figures, in us, are those of the
// kernels' own timelines; one or two one-tile blocks share a multiprocessor.  Measured, us: 17 tokens behind 500 in a cluster 8.5, with join_kernel 9.0; 32 behind
// 500, INT8, 9.6 and 11.8; 100 of 32 kv heads behind 400 9.8 and 12.1; 24 behind 60000 one block per multiprocessor 72, two 43.6; 8 sequences behind 1024 shared
// positions two 19.2, one 8.4.  Rounds left whole and with the rest split: 4096 tokens behind 12000 (3.5 rounds) 923 and 888 (in a row, at the power limit), 1500
// behind 6000 201 and 159, 1200 of 32 kv heads behind 30000 (160 blocks) 904 and 620.  Not, when this was chosen, for small gains over sequences of unequal length,
// whose last round is short anyway (six portions of 250: 64.4 and 68.7); nor all items of several rounds (81.8), nor clusters of two blocks per multiprocessor (four
// of 20 behind 8000, INT8: 37.4, join_kernel 34.5).
struct Plan {
  int tiles, row_blocks, nsplit, cluster, parts;
  long long items, split;  // (rows of a block, kv head) pairs; the last so many of them are split
  long long split_rows(long long all) const { return split == items ? all : split * tiles * kRows; }
};
constexpr float kTwoTilesPage = 0.92f, kTwoTilesFixed = 5.5f;  // us
Plan plan_tiles(long long rows, int batch, long long num_rows, int kv_heads, long long pages, bool prompt) {
  constexpr float kJoinCluster = 1.f, kJoinKernel = 4.f, kJoinTail = 0.1f, kPartBytesPerUs = 1e7f;
  Plan pl{};
  pl.tiles = rows <= kRows ? 1 : 2;
  const long long block_rows = pl.tiles * kRows, sms = num_sms();
  pl.row_blocks = static_cast<int>((rows + block_rows - 1) / block_rows);
  pl.items = static_cast<long long>(pl.row_blocks) * batch * kv_heads;
  // blocks that have rows: of portions of unequal length the shorter ones leave some without
  long long blocks = static_cast<long long>(kv_heads) * ((2 * num_rows + batch * block_rows + 2 * block_rows - 1) / (2 * block_rows));
  blocks = blocks < 1 ? 1 : blocks > pl.items ? pl.items : blocks;
  const unsigned most = static_cast<unsigned>(pages < 1 ? 1 : pages);
  const float fixed = pl.tiles == 2 ? kTwoTilesFixed : 3.5f;
  float best = 3.0e38f;
  auto take = [&](float t, unsigned n, unsigned cluster, long long split) {
    if (t >= best) return;
    best = t;
    pl.nsplit = static_cast<int>(n);
    pl.cluster = static_cast<int>(cluster);
    pl.split = split;
  };
  for (int per_sm = 1; per_sm <= (pl.tiles == 1 ? 2 : 1); ++per_sm) {
    const float page = pl.tiles == 2 ? kTwoTilesPage : per_sm == 1 ? (rows <= 64 ? 0.7f : 0.95f) : (rows <= 64 ? 1.f : 1.2f);
    const long long slots = sms * per_sm;
    auto block = [&](unsigned n) { return ((most + n - 1) / n) * page + fixed; };
    // sequences of a batch differ in length, and the blocks of the last round are short beside the longest: half of what it lacks to be full
    auto rounds = [&](long long of) {
      const float full = static_cast<float>((of + slots - 1) / slots);
      return batch == 1 || of <= slots ? full : 0.5f * (full + of / static_cast<float>(slots));
    };
    auto join = [&](long long split, unsigned n) {
      return prompt ? kJoinKernel + (split * (num_rows * kv_heads / static_cast<float>(blocks)) * n) * (2.f * (kD * 4 + 8)) / kPartBytesPerUs : kJoinTail * n;
    };
    take(rounds(blocks) * block(1), 1, 1, prompt ? 0 : pl.items);
    // splits of one round
    const long long room = slots / blocks;
    const unsigned last = static_cast<unsigned>(room > 128 ? 128 : room);
    for (unsigned n = per_sm == 1 || sms < blocks ? 2 : static_cast<unsigned>(sms / blocks) + 1; n <= last && n <= most; ++n) {
      const bool cluster = prompt && pl.tiles == 1 && per_sm == 1 && n <= kMostCluster && (n & (n - 1)) == 0;
      take(block(n) + (cluster ? kJoinCluster : join(pl.items, n)), n, cluster ? n : 1, pl.items);
    }
    // whole rounds, and splits of the rest
    for (long long whole = blocks / slots; prompt && whole >= 1 && whole + 1 >= blocks / slots; --whole) {
      const long long rest = blocks - whole * slots;
      const float of_doubt = batch == 1 ? 1.f : 1.1f;
      for (unsigned n = 2; rest > 0 && n <= 8 && n <= most; ++n) take((whole * block(1) + rounds(rest * n) * block(n) + join(rest, n)) * of_doubt, n, 1, rest);
    }
  }
  pl.parts = pl.nsplit / pl.cluster;
  return pl;
}
size_t part_bytes(long long rows, int parts) { return static_cast<size_t>(rows) * parts * (kD * sizeof(float) + sizeof(float2)); }

template <int BITS, int TILES, int MODE>
int run_tiles(const TileParams& p, long long blocks, void* stream) {
  using C = TileCfg<BITS, TILES>;
  const int rc = allow_smem<tile_kernel<BITS, TILES, MODE>>(C::kSmem, "paged attention: shared memory", [](int regs) { return !C::kShares || shares_suffice(regs); });
  if (rc) return rc;
  QS_REQUIRE(blocks <= 0x7fffffffll, "paged attention: %lld blocks", blocks);
  return launch(tile_kernel<BITS, TILES, MODE>, dim3(static_cast<unsigned>(blocks)), C::kThreads, C::kSmem, stream, "paged attention", p.cluster, p);
}
int tiles(TileParams& p, const Plan& pl, bool int4, void* stream) {
  p.row_blocks = pl.row_blocks; p.nsplit = pl.nsplit; p.cluster = pl.cluster; p.parts = pl.parts;
  p.split_from = static_cast<int>(pl.items - pl.split); p.block_rows = pl.tiles * kRows; p.run = p.split_from ? static_cast<int>(pl.split) : p.num_kv_heads;
  const long long blocks = pl.items + pl.split * (pl.nsplit - 1);
  auto sized = [&](auto bits) {
    constexpr int kBits = decltype(bits)::value;
    if (pl.tiles == 2) return p.part ? run_tiles<kBits, 2, kPartial>(p, blocks, stream) : run_tiles<kBits, 2, kWhole>(p, blocks, stream);
    if (pl.cluster > 1) return run_tiles<kBits, 1, kCluster>(p, blocks, stream);
    return p.part ? run_tiles<kBits, 1, kPartial>(p, blocks, stream) : run_tiles<kBits, 1, kWhole>(p, blocks, stream);
  };
  return int4 ? sized(std::integral_constant<int, 4>{}) : sized(std::integral_constant<int, 8>{});
}

Plan plan_prompt(int batch, int num_tokens, int max_seqlen, int max_length, int heads, int kv_heads) {
  const int group = heads / kv_heads;
  return plan_tiles(static_cast<long long>(max_seqlen) * group, batch, static_cast<long long>(num_tokens) * group, kv_heads,
                    (static_cast<long long>(max_length) + kPage - 1) / kPage, true);
}
// Few sequences or few shared pages: the tail kernel reads the shared pages too, once per sequence (out of the first row of the table), one launch instead of two.
// us, both kernels / the tail alone (INT4, 32 heads over 8, 100 positions behind): one sequence behind 512 6.7 / 6.0, behind 4096 9.6 / 8.2; two behind 512 6.8 / 6.1;
// eight behind 128 7.5 / 4.9.  With 8 kv heads more would gain (two behind 2048 8.3 / 7.1, eight behind 512 7.7 / 7.1), with 32 no longer (eight behind 512 9.3 /
// 10.5).
bool tail_alone(int batch, int shared_blocks) { return batch == 1 || static_cast<long long>(batch) * shared_blocks <= 16; }
Plan plan_shared(int batch, int shared_blocks, int heads, int kv_heads) {
  const long long rows = static_cast<long long>(batch) * (heads / kv_heads);
  return plan_tiles(rows, 1, rows, kv_heads, shared_blocks, false);
}

}  // namespace

size_t paged_prompt_workspace(int batch, int num_tokens, int max_seqlen, int max_length, int heads, int kv_heads) {
  if (batch <= 0 || num_tokens <= 0 || max_seqlen <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
  const Plan pl = plan_prompt(batch, num_tokens, max_seqlen < num_tokens ? max_seqlen : num_tokens, max_length, heads, kv_heads);
  return pl.parts > 1 ? part_bytes(pl.split_rows(static_cast<long long>(num_tokens) * heads), pl.parts) : 0;
}

int paged_prompt_attention(const PagedAttnArgs& a) {
  if (a.batch == 0 || a.num_tokens == 0 || a.max_seqlen == 0) return QS_OK;
  const Plan pl = plan_prompt(a.batch, a.num_tokens, a.max_seqlen, a.max_length, a.num_heads, a.cache.num_kv_heads);
  TileParams p{};
  p.q = static_cast<const __half*>(a.q); p.out = static_cast<__half*>(a.out); p.q_stride = a.q_stride; p.out_stride = a.out_stride;
  p.kv_pointers = a.cache.kv_pointers; p.cu = a.cache.cu_seqlens; p.lengths = a.cache.lengths;
  p.batch = a.batch; p.num_tokens = a.num_tokens; p.max_seqlen = a.max_seqlen; p.max_blocks = a.cache.max_blocks; p.num_heads = a.num_heads; p.num_kv_heads = a.cache.num_kv_heads;
  p.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  const long long rows = pl.split_rows(static_cast<long long>(a.num_tokens) * a.num_heads);
  if (pl.parts > 1) {
    QS_REQUIRE(a.workspace && a.workspace_bytes >= part_bytes(rows, pl.parts), "paged_prompt_attention: workspace of %zu bytes, %zu needed", a.workspace_bytes,
               part_bytes(rows, pl.parts));
    QS_REQUIRE(rows <= 0x7fffffffll, "paged_prompt_attention: %lld rows", rows);
    p.part = static_cast<float*>(a.workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part + rows * pl.parts * kD);
  }
  const int rc = tiles(p, pl, a.cache.int4, a.stream);
  if (rc || pl.parts == 1) return rc;
  const bool wide = pl.parts >= 8;  // (24 tokens behind 60000, 37 parts: a warp a row 44.3 us, four 43.6; 4 behind 4000 10.9 and 9.9; 1500 behind 6000, a few: 160 and 175)
  return launch(wide ? join_kernel<4> : join_kernel<1>, dim3(static_cast<unsigned>(wide ? rows : (rows + 3) / 4)), 128, 0, a.stream, "paged_prompt_attention: join", 1, p);
}

size_t shared_prefix_workspace(int batch, int shared_blocks, int heads, int kv_heads) {
  if (batch <= 0 || shared_blocks <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || tail_alone(batch, shared_blocks)) return 0;
  return part_bytes(static_cast<long long>(batch) * heads, plan_shared(batch, shared_blocks, heads, kv_heads).parts);
}

// The tail kernel's blocks start while the prefix's run, on the multiprocessors that those leave, as many on each as it holds.  (Blocks of two tiles leave no room
// beside them; one-tile blocks do.)  So where the tail's fit, fewer splits of the prefix and a bound on the tail's blocks per multiprocessor let both end at about the
// same time. Chooses the splits, no more than planned, and returns that bound; one behind the other, the bound spreads the tail evenly.  The tail's estimate, us:
// start and join, that of its blocks' issue slots, and its warps' half pages, each its own chain or its share of the issue slots.  Measured, one behind the other /
// side by side, 8 kv heads: 38 sequences, 500 positions behind 1024, 20.1 / 12.5 (INT8 18.3 / 12.9); 64, 1000 behind 2048, 29.0 / 24.8; bounded alone: 38, 1000 behind
// 16384, 40.3 / 37.1.  Not for small estimated gains (INT8, 38, 200 behind 4096: 18.5 / 21.6).
int side_by_side(Plan& pl, int shared_blocks, long long tail, long long tail_pages, int cluster, int most) {
  const long long sms = num_sms(), even = (tail + sms - 1) / sms;
  if (pl.tiles == 1 || even > most) return most;
  const int steps = static_cast<int>(tail_pages > 0 ? (2 * tail_pages + kTailWarps * cluster - 1) / (kTailWarps * cluster) : 0);
  auto prefix = [&](long long n) { return ((shared_blocks + n - 1) / n) * kTwoTilesPage + kTwoTilesFixed; };
  auto own = [&](long long k) {
    const float busy = (most == 4 ? 0.4f : 0.45f) * k;
    return 3.f + 1.1f * k + steps * (busy > 0.9f ? busy : 0.9f);
  };
  int room = static_cast<int>(even);
  float best = 0.85f * (prefix(pl.nsplit) + own(even));
  long long splits = pl.nsplit;
  for (int k = 1; k <= most; ++k) {
    long long n = (sms - (tail + k - 1) / k) / pl.items;
    n = n < pl.nsplit ? n : pl.nsplit;
    if (n < 1) continue;
    const float t = prefix(n) > own(k) ? prefix(n) : own(k);
    if (t < best) {
      best = t;
      splits = n;
      room = k;
    }
  }
  pl.nsplit = pl.parts = static_cast<int>(splits);
  return room;
}

int shared_prefix_attention(const PagedAttnArgs& a, int shared_blocks) {
  if (a.batch == 0) return QS_OK;
  TailParams t{};
  if (tail_alone(a.batch, shared_blocks)) {
    t.common = shared_blocks;
    shared_blocks = 0;
  }
  const long long rows = static_cast<long long>(a.batch) * a.num_heads;
  t.q = static_cast<const __half*>(a.q); t.out = static_cast<__half*>(a.out); t.q_stride = a.q_stride; t.out_stride = a.out_stride;
  t.batch = a.batch; t.kv_pointers = a.cache.kv_pointers; t.lengths = a.cache.lengths; t.max_blocks = a.cache.max_blocks; t.num_heads = a.num_heads;
  t.num_kv_heads = a.cache.num_kv_heads; t.shared_blocks = shared_blocks; t.scale_log2 = a.softmax_scale * 1.4426950408889634f;
  const int group = a.num_heads / t.num_kv_heads, heads_y = t.num_kv_heads * ((group + kMaxG - 1) / kMaxG);
  // shares of a sequence's pages: as many blocks as the device holds at a time, a page for each warp pair at least
  const int most = a.cache.int4 ? 4 : 3;  // blocks per multiprocessor
  const long long sms = num_sms(), slots = sms * most, blocks = static_cast<long long>(heads_y) * a.batch;
  const long long tail_pages = (static_cast<long long>(a.max_length) + kPage - 1) / kPage - shared_blocks;
  t.cluster = 1;
  while (t.cluster < kMaxCluster && blocks * t.cluster * 2 <= slots && tail_pages >= 2 * kTailWarps * t.cluster) t.cluster *= 2;
  QS_REQUIRE(blocks <= 0x7fffffffll, "shared_prefix_attention: %lld runs of heads", blocks);
  const bool shared = blocks < 12 * num_sms();  // (a wave of warps; 128 sequences x 32 heads, INT8, up to 511 positions each behind 16384: 155 us by blocks, 127 by warps)
  if (!shared) t.cluster = 1;
  int room = most;
  if (shared_blocks > 0) {
    Plan pl = plan_shared(a.batch, shared_blocks, a.num_heads, a.cache.num_kv_heads);
    QS_REQUIRE(a.workspace && a.workspace_bytes >= part_bytes(rows, pl.parts), "shared_prefix_attention: workspace of %zu bytes, %zu needed", a.workspace_bytes,
               part_bytes(rows, pl.parts));
    if (shared) room = side_by_side(pl, shared_blocks, blocks * t.cluster, tail_pages, t.cluster, most);
    TileParams p{};
    p.q = t.q; p.q_stride = t.q_stride; p.kv_pointers = t.kv_pointers; p.lengths = t.lengths;
    p.batch = 1; p.num_tokens = p.max_seqlen = a.batch; p.max_blocks = t.max_blocks; p.num_heads = t.num_heads; p.num_kv_heads = t.num_kv_heads;
    p.shared_blocks = shared_blocks; p.scale_log2 = t.scale_log2;
    p.part = static_cast<float*>(a.workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part + rows * pl.parts * kD);
    t.nsplit = pl.parts; t.part = p.part; t.part_ml = p.part_ml;
    const int rc = tiles(p, pl, a.cache.int4, a.stream);
    if (rc) return rc;
  }
  const dim3 grid = shared ? dim3(t.cluster, heads_y, a.batch) : dim3(static_cast<unsigned>((blocks + kTailWarps - 1) / kTailWarps));
  // us, two slots / four (INT4): one sequence of 16384 positions 17.6 / 16.2, one of 2000 with 32 heads a group of one 8.1 / 6.2, four of up to 8000 17.3 / 12.1.  Not
  // behind the tile kernel, whose blocks leave no room for it: 32 sequences, 100 positions behind 4096, 13.1 / 15.8
  const bool deep = shared && t.nsplit == 0 && blocks * t.cluster <= 2 * num_sms();
  auto run = [&](auto bits, auto by_block, auto more) {
    constexpr int kBits = decltype(bits)::value;
    constexpr bool kShared = decltype(by_block)::value, kDeep = decltype(more)::value;
    constexpr int kSm = 228 * 1024, kOwn = SliceCfg<kBits, kDeep>::kSmem;
    const int rc = allow_smem<tail_kernel<kBits, kShared, kDeep>>(kOwn > kSm / 2 ? kOwn : kSm / 2, "shared_prefix_attention: shared memory", [](int) { return true; });
    if (rc) return rc;
    const int smem = room < most && kOwn < kSm / (room + 1) ? kSm / (room + 1) : kOwn;  // so much that no more than `room` blocks share a multiprocessor
    return launch(tail_kernel<kBits, kShared, kDeep>, grid, 32 * kTailWarps, smem, a.stream, "shared_prefix_attention", t.cluster, t);
  };
  auto with = [&](auto bits) {
    if (!shared) return run(bits, std::false_type{}, std::false_type{});
    return deep ? run(bits, std::true_type{}, std::true_type{}) : run(bits, std::true_type{}, std::false_type{});
  };
  return a.cache.int4 ? with(std::integral_constant<int, 4>{}) : with(std::integral_constant<int, 8>{});
}

}  // namespace qs
