// qserve_b200 -- drafted tokens of a step: what the rows of a tree see of one another, and their verification against the target's probabilities.
//
// The rows of sequence b are a portion (as in paged_cache.cu): row 0 the token that the step starts from, every other one a drafted token with a parent
// among the rows ahead of it.  Row i's logits are the target's behind row i, so they decide on i's children.
//
// verify, of a sequence with temperature t > 0 (p = softmax(logits / t) of the current row, from row 0 on):
//   drafts drawn from q, a chain:  the child x is taken where u q(x) < p(x); else the sequence ends with a token drawn from max(p - q, 0) / sum;
//   drafts as they come, a tree:   the first child x_j with u < p(x_1) + ... + p(x_j) (a token counts once); else a token drawn from p without the children;
//   no child:                      a token drawn from p.
// Either way the tokens are distributed as if they were drawn from the target one by one.  A token is drawn at r as the first one whose running sum is above r times
// the whole.  t = 0: the child with the row's largest logit; the lowest index of equal ones.
#include <cuda_bf16.h>
#include <math_constants.h>

#include "common.cuh"
#include "launch.h"
#include "paged_common.cuh"

namespace qs {
namespace {

using paged::Portion;
using paged::portion_of;

// ------------------------------------------------------------------------------------------------------------------------
// tree: thread = row, up the ancestors, one load of shared memory behind the other.  A launch with next to nothing behind it: 128 trees of up to 64 rows 4.3 us, one of 26
// rows 4.3, where an empty kernel takes 2 and the loads of starts, lengths and parents one after the other the rest.
// ------------------------------------------------------------------------------------------------------------------------
constexpr int kWords = kMostDrafted / 64;

__global__ void __launch_bounds__(kMostDrafted) tree_kernel(int* positions, unsigned long long* visible, const int* parents, const int* cu, const int* lengths, int num_tokens,
                                                            int max_seqlen, int words) {
  __shared__ int s_parent[kMostDrafted];
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.x, i = threadIdx.x;
  const Portion portion = portion_of(cu, lengths, b, num_tokens);
  const int n = min(portion.count, max_seqlen);
  if (i < n) s_parent[i] = parents[portion.start + i];
  __syncthreads();
  if (i >= n) return;
  unsigned long long seen[kWords] = {};
  int at = i, depth = 0;
  while (at > 0) {  // a parent lies ahead of its child, so this ends
    const int up = s_parent[at];
    if (up < 0 || up >= at) break;  // padding
#pragma unroll
    for (int w = 0; w < kWords; ++w) seen[w] |= w == at >> 6 ? 1ull << (at & 63) : 0ull;
    at = up;
    ++depth;
  }
  if (at == 0) seen[0] |= 1ull;
  positions[portion.start + i] = portion.first + depth;
#pragma unroll
  for (int w = 0; w < kWords; ++w)
    if (w < words) visible[static_cast<long long>(portion.start + i) * words + w] = seen[w];
}

// ------------------------------------------------------------------------------------------------------------------------
// verification: a cluster per sequence, its warps side by side over the vocabulary
//
// Every row that the walk may need is read once for its maximum and sum of exponentials in 32 bits, a window of rows at a time: the current one and those behind it if
// every first child is taken.  Blocks exchange maxima and sums through one another's shared memory, and each warp decides one row of the window.  A decision that 32
// bits could get wrong is taken again with a sum of 64 bits.  The token that the sequence ends with is drawn with weights and sums of 64 bits: among 10^5 tokens one
// border or another lies within 32 bits' error of one draw in a hundred.  For that the last row is read once more, out of L2.
//
// 64 chains of up to 6 rows with the draft's probabilities, 128256 tokens, fp16, two blocks a chain: 45.5 us, of which maxima and sums take 19 (77 MB, 4.1 TB/s of 128
// multiprocessors' copies), the second reading of a row and its probabilities 14 (48 MB; 46 cycles of the 64-bit pipe for a warp's 32 numbers), exchanges and decisions 4,
// the search for the drawn token 3.5, start and end 4; over all of it issue slots are at 0.47, the 64-bit pipe at 0.14.  Few sequences wait for one another's blocks
// instead: one chain of 5, 32000 tokens, 13.4, a quarter of it for instructions.  Blocks of 8 warps, two on a multiprocessor, 51.7 (of 46.5 then).
// ------------------------------------------------------------------------------------------------------------------------
constexpr int kVerifyWarps = 16, kVerifyThreads = 32 * kVerifyWarps, kMostBlocks = 16;
constexpr int kMostWindow = 8;
constexpr int kSteps = 32;  // of an octave, in the table of powers of two
// Words of 16 bytes of a lane: so many are copied to shared memory and taken out of it together, and so many such groups are on their way, 128 KB a multiprocessor.
// (What registers hold, four words, leaves it at 2.7 TB/s over the device.)  A lane reads what it has copied itself, so nothing waits but its own copies.
constexpr int kGroup = 4, kStages = 4, kDepth = kGroup * kStages;
constexpr int kRingBytes = kVerifyWarps * kDepth * 512;
static_assert(kVerifyThreads >= kMostDrafted && kSteps <= 32 && kVerifyWarps >= kMostWindow && kVerifyWarps >= kMostBlocks, "a thread per row, a warp per row of a window");

template <typename T>
__device__ __forceinline__ float number(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(x);
  else return __bfloat162float(x);
}
// two numbers of one 32-bit word (16-bit types; whole words at a time, or the compiler takes them apart by byte), or one
template <typename T>
__device__ __forceinline__ float2 pair_of(uint32_t w) {
  if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// a 16-byte word's numbers
template <typename T, int N>
__device__ __forceinline__ void numbers_of(const uint4& w, float (&x)[N]) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (N == 4) {
      x[i] = __uint_as_float(words[i]);
    } else {
      const float2 two = pair_of<T>(words[i]);
      x[2 * i] = two.x;
      x[2 * i + 1] = two.y;
    }
  }
}
// the largest of a word's numbers; what is no number is passed over
template <typename T>
__device__ __forceinline__ float largest_of(const uint4& w) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* x = reinterpret_cast<const T2*>(&w);
    const T2 m = __hmax2(__hmax2(x[0], x[1]), __hmax2(x[2], x[3]));
    return fmaxf(number(m.x), number(m.y));
  }
}

// A row of logits in 16-byte words: word c holds the numbers kN c - skip .. + kN - 1.  The first and the last word may reach past the row; those between are copied as they
// lie.
template <typename T>
struct Row {
  static constexpr int kN = 16 / sizeof(T);
  const T* p;
  int skip, vocab, words;
  __device__ __forceinline__ Row(const T* row, int v) : p(row), vocab(v) {
    skip = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    words = (skip + v + kN - 1) / kN;
  }
  __device__ __forceinline__ int first(int c) const { return c * kN - skip; }
  __device__ __forceinline__ bool whole(int c) const { return first(c) >= 0 && first(c) + kN <= vocab; }
  __device__ __forceinline__ const uint4* at(int c) const { return reinterpret_cast<const uint4*>(p - skip) + c; }
  // of the words w0 .. w1 - 1 those that are whole: b0 .. b1 - 1
  __device__ __forceinline__ int whole_from(int w0, int w1) const { return w0 < w1 && !whole(w0) ? w0 + 1 : w0; }
  __device__ __forceinline__ int whole_to(int b0, int w1) const { return b0 < w1 && !whole(w1 - 1) ? w1 - 1 : w1; }
  // -inf for what lies outside the row
  __device__ __forceinline__ uint4 word(int c) const { return whole(c) ? __ldcg(at(c)) : edge(p, first(c), vocab); }
  static __device__ __noinline__ uint4 edge(const T* p, int first, int vocab) {
    uint4 r;
    T* t = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const int i = first + k;
      if (i >= 0 && i < vocab) t[k] = p[i];
      else t[k] = static_cast<T>(-CUDART_INF_F);
    }
    return r;
  }
};

struct VerifyParams {
  const void* logits;
  long long logits_stride, probs_stride;
  const long long* tokens;
  const int* parents;
  const float* probs;
  const int* cu;
  const float *coins, *draws, *temperatures;
  long long* out_tokens;
  int *out_rows, *out_counts;
  int num_tokens, vocab, max_seqlen, cluster, per_block, per_warp, window;  // per_block: a row's words of each block of the cluster, of each of its warps; the last ones' are fewer
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t peer_of(const void* mine, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
  return a;
}
__device__ __forceinline__ void put_peer(const double* mine, uint32_t rank, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(peer_of(mine, rank)), "d"(v) : "memory"); }
__device__ __forceinline__ void put_peer(const uint2* mine, uint32_t rank, uint2 v) {
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(peer_of(mine, rank)), "r"(v.x), "r"(v.y) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ uint4 take16(uint32_t from) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
  return v;
}
// Copies of a lane that may still be on their way when it goes on
template <int PENDING>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// What a number weighs against its row's largest one, in 64 bits: exp((x - top) / t) = 2^(-y / 32), y = (top - x) 32 log2(e) / t, as 2^(-n / 32) from the table times
// 1 + g + g^2 / 2 + g^3 / 6 + g^4 / 24 of the rest |g| <= ln(2) / 64: off by g^5 / 120 = 1.2e-12 of itself at most.  Nine operations of 64 bits, where exp() has about
// 25; a table of 32 entries meets every bank of shared memory twice at most.  (A larger table and one product less took longer.)
struct Weigh {
  double per_unit, span;  // 32 log2(e) / t; 2^14 of those
  double top;
  uint32_t power;        // 2^(i / 32), in shared memory
  float least;           // what is above it weighs 2^-512 at least
  bool odd;              // the largest has no end, and those without one share the weight; or there is no number to take for all that weigh nothing
  __device__ __forceinline__ void against(float largest) {
    top = largest;
    least = __double2float_rd(top - fmax(span, fabs(top) * 1e-12));  // y below 2^14; a number below top in any case
    odd = !((top - static_cast<double>(least)) * per_unit < 30000.0);  // (2^-1022 is 2^(-32704 / 32))
  }
  __device__ __forceinline__ double finite(float x) const {
    const double d = top - static_cast<double>(x);
    constexpr double kMagic = 6755399441055744.0;  // 1.5 x 2^52: a sum with it has a whole number in its low bits
    const double z = fma(d, -per_unit, kMagic), g = fma(d, -per_unit, kMagic - z);
    const int n = __double2loint(z);  // -y, rounded
    constexpr double c1 = 0.02166084939249829, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6, c4 = c1 * c1 * c1 * c1 / 24;  // ln(2) / 32
    double m;
    asm("ld.shared.f64 %0, [%1];" : "=d"(m) : "r"(power + ((n << 3) & (8 * kSteps - 8))));
    const double e = fma(m, g * fma(g, fma(g, fma(g, c4, c3), c2), c1), m);
    return __hiloint2double(__double2hiint(e) + ((n >> 5) << 20), __double2loint(e));
  }
  // 0 for what is no number, or weighs less than that
  __device__ __forceinline__ double operator()(float x) const {
    if (top == CUDART_INF_F) return x == CUDART_INF_F ? 1.0 : 0.0;
    return x > least ? finite(x) : 0.0;
  }
  // the same of a word; but 2^-512 in place of 0 where the row is not odd: kNothing is above what a vocabulary of those weighs
  template <bool ODD, typename T, int N>
  __device__ __forceinline__ void word(const uint4& its, double (&w)[N]) const {
    float x[N];
    numbers_of<T>(its, x);
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = ODD ? (*this)(x[k]) : finite(fmaxf(x[k], least));
  }
};
constexpr double kNothing = 1e-140;

// What a lane's share of a row's words w0 .. w1 - 1 weighs: in all; what is drawn from it, with S = `total` the row's sum as far as it is known, e - S q where that is
// above 0 (Q), or e without the `kids`; and the draft's share q of the numbers drawn from.  (A function of its own: inlined where it is called the kernel waits for
// instructions.)
struct Shares {
  double all, drawn;
  float draft;
};
template <typename T, bool Q, bool ODD>
__device__ __noinline__ Shares shares_of(const T* p, int vocab, int w0, int w1, const float* q, double total, Weigh weigh, const int* kids, int num_kids) {
  constexpr int kN = Row<T>::kN, kAhead = 2;
  const Row<T> row(p, vocab);
  const int lane = threadIdx.x & 31;
  Shares sum{0.0, 0.0, 0.f};
  auto add = [&](int c, const uint4& its, const float (&qs)[kN]) {
    double w[kN];
    weigh.word<ODD, T>(its, w);
#pragma unroll
    for (int k = 0; k < kN; ++k) sum.all += w[k];
    if constexpr (Q) {
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        const double d = fma(-total, static_cast<double>(qs[k]), w[k]);
        asm("{\n\t.reg .pred p;\n\tsetp.ge.s32 p, %2, 0;\n\t@p add.f64 %0, %0, %3;\n\t@p add.f32 %1, %1, %4;\n\t}"  // not below zero
            : "+d"(sum.drawn), "+f"(sum.draft)
            : "r"(__double2hiint(d)), "d"(d), "f"(qs[k]));
      }
    } else if (num_kids > 0) {
      for (int j = 0; j < num_kids; ++j) {
        const int i = kids[j] - row.first(c);
#pragma unroll
        for (int k = 0; k < kN; ++k)
          if (k == i) w[k] = 0.0;
      }
#pragma unroll
      for (int k = 0; k < kN; ++k) sum.drawn += w[k];
    }
  };
  // The whole words, two of a lane on their way while one is taken.  q's words of four begin where the row's words do, or its numbers are loaded one by one.
  const bool wide = Q && (reinterpret_cast<uintptr_t>(q - row.skip) & 15) == 0;
  const int b0 = row.whole_from(w0, w1), b1 = row.whole_to(b0, w1);
  uint4 its[kAhead + 1];
  float qs[kAhead + 1][kN];
  auto load = [&](int c, uint4& word, float (&of_q)[kN]) {
    if (c >= b1) return;
    word = __ldcg(row.at(c));
    if constexpr (Q) {
      const float* const from = q + row.first(c);
      if (wide) {
#pragma unroll
        for (int k = 0; k < kN; k += 4) {
          const float4 four = __ldcg(reinterpret_cast<const float4*>(from + k));
          of_q[k] = four.x; of_q[k + 1] = four.y; of_q[k + 2] = four.z; of_q[k + 3] = four.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < kN; ++k) of_q[k] = __ldcg(from + k);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) load(b0 + lane + 32 * i, its[i], qs[i]);
#pragma unroll 1
  for (int c = b0 + lane; c < b1; c += 32) {
    load(c + 32 * kAhead, its[kAhead], qs[kAhead]);
    add(c, its[0], qs[0]);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      its[i] = its[i + 1];
#pragma unroll
      for (int k = 0; k < kN; ++k) qs[i][k] = qs[i + 1][k];
    }
  }
  if (lane == 0 ? b0 > w0 : lane == 1 && b1 < w1) {  // the others, a lane each
    const int c = lane == 0 ? w0 : w1 - 1;
#pragma unroll
    for (int k = 0; k < kN; ++k) qs[0][k] = Q && row.first(c) + k >= 0 && row.first(c) + k < vocab ? q[row.first(c) + k] : 0.f;
    add(c, row.word(c), qs[0]);
  }
  __syncwarp();
  if (!Q && num_kids == 0) sum.drawn = sum.all;
  return sum;
}

// all threads of a cluster
__device__ __forceinline__ void meet_of(int cluster) {
  if (cluster > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
}

// A token drawn from max(e - S q, 0), number by number, S = `all` the row's sum of 64 bits; where that leaves nothing, from the weights e.  A run of the row for each of
// the cluster's warps; the one that the threshold falls into shared out over its block's lanes.  `of_warps`, `of_blocks`: places for sums, the blocks' twice.  (A function
// of its own, with nothing to come back to but the end: the pass above once more, in a loop or called again, held registers that made 64 chains of 6, 128256 tokens, 1 to
// 3 us longer where none needs it.  Where all do, 64 rows of 128256 tokens and their q take 64 us, 32 without it; one row of 32000 15, 12.4 without.  A run of the row for
// each thread of the cluster, in place of the two steps: 123 us, for loads that lie apart.)
template <typename T>
__device__ __noinline__ void draw_exactly(const T* p, int vocab, const float* q, double all, Weigh weigh, float draw, double* of_warps, double* of_blocks0, double* of_blocks1, int cluster, int rank,
                                          long long* out) {
  constexpr int kN = Row<T>::kN;
  const Row<T> row(p, vocab);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the sum over words c0, c0 + step, .. ahead of c1; or the first number with which the sum from `ahead` on is past the threshold, the last with any weight if none is
  auto go_through = [&](int c0, int c1, int step, bool search, double ahead, double threshold, int& found) {
    double sum = 0.0;
#pragma unroll 1
    for (int c = c0; c < c1; c += step) {
      float x[kN], qs[kN];
      const int first = row.first(c);
#pragma unroll
      for (int k = 0; k < kN; ++k) qs[k] = q && static_cast<unsigned>(first + k) < static_cast<unsigned>(vocab) ? __ldcg(q + first + k) : 0.f;
      numbers_of<T>(row.word(c), x);
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        double w = weigh(x[k]);
        if (q) w = w > 0.0 ? fma(-all, static_cast<double>(qs[k]), w) : 0.0;
        if (!(w > 0.0)) continue;  // (what lies outside the row among them)
        sum += w;
        if (!search) continue;
        found = first + k;
        if (ahead + sum > threshold) return sum;
      }
    }
    return sum;
  };
  auto run_of = [&](double x) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double below = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += below;
    }
    return x;
  };
  const int per_warp = (row.words + kVerifyWarps * cluster - 1) / (kVerifyWarps * cluster);
  auto begin_of = [&](int w) { return static_cast<int>(min(static_cast<long long>(row.words), static_cast<long long>(per_warp) * w)); };
  int found = -1;
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const int mine = rank * kVerifyWarps + warp;
    const double of_mine = run_of(go_through(begin_of(mine) + lane, begin_of(mine + 1), 32, false, 0.0, 0.0, found));
    double* const of_blocks = pass == 0 ? of_blocks0 : of_blocks1;
    __syncthreads();  // what lay in the places has been read
    if (lane == 31) of_warps[warp] = of_mine;
    __syncthreads();
    const double of_warp = lane < kVerifyWarps ? of_warps[lane] : 0.0, run_warps = run_of(of_warp);
    if (warp == 0) {
      const double of_block = __shfl_sync(0xffffffffu, run_warps, 31);
      if (cluster == 1) of_blocks[0] = of_block;
      else if (lane < cluster) put_peer(&of_blocks[rank], lane, of_block);
    }
    meet_of(cluster);
    const double of_block = lane < cluster ? of_blocks[lane] : 0.0, run_blocks = run_of(of_block), whole = __shfl_sync(0xffffffffu, run_blocks, 31);
    if (q && !(whole > 0.0)) {  // all blocks alike
      q = nullptr;
      continue;
    }
    const double threshold = static_cast<double>(draw) * whole;
    double ahead = 0.0;
    auto choose = [&](double share, double run) {
      const unsigned any = __ballot_sync(0xffffffffu, share > 0.0), past = __ballot_sync(0xffffffffu, share > 0.0 && ahead + run > threshold);
      const int chosen = past ? __ffs(past) - 1 : 31 - __clz(any);
      ahead += __shfl_sync(0xffffffffu, run - share, chosen & 31);
      return chosen;
    };
    if (choose(of_block, run_blocks) != rank) return;  // the whole block
    const int in = rank * kVerifyWarps + choose(of_warp, run_warps), w0 = begin_of(in), len = begin_of(in + 1) - w0;
    const int c0 = w0 + static_cast<int>(static_cast<long long>(len) * threadIdx.x / kVerifyThreads), c1 = w0 + static_cast<int>(static_cast<long long>(len) * (threadIdx.x + 1) / kVerifyThreads);
    const double of_lane = go_through(c0, c1, 1, false, 0.0, 0.0, found), run_lanes = run_of(of_lane);
    __syncthreads();  // of_warps has been read
    if (lane == 31) of_warps[warp] = run_lanes;
    __syncthreads();
    const double of_run = lane < kVerifyWarps ? of_warps[lane] : 0.0;
    if (choose(of_run, run_of(of_run)) == warp && choose(of_lane, run_lanes) == lane) {
      go_through(c0, c1, 1, true, ahead, threshold, found);
      *out = found;
    }
    return;
  }
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const __grid_constant__ VerifyParams p) {
  constexpr int kN = Row<T>::kN;
  extern __shared__ __align__(16) uint4 s_ring[];
  __shared__ double s_power[kSteps];
  // sums of 64 bits over a row's weights: all of them; those that a token is drawn from, with the draft's share as the sum of 32 bits has it; the draft's
  __shared__ double s_share[3][kVerifyWarps], s_shares[2][3][kMostBlocks];
  __shared__ uint2 s_part[kMostWindow][kVerifyWarps + 1];            // a row's maximum, and sum or word: of the warps, and of the words that reach past the row
  __shared__ uint2 s_all[2][kMostWindow][kMostBlocks];               // of the blocks
  __shared__ int s_parent[kMostDrafted], s_token[kMostDrafted], s_first[kMostDrafted], s_path[kMostDrafted], s_kids[kMostDrafted];
  __shared__ float s_x[kMostDrafted], s_q[kMostDrafted], s_coin[kMostDrafted];
  __shared__ unsigned char s_again[kMostDrafted];
  __shared__ int s_next[kMostWindow], s_largest[kMostWindow], s_num_kids, s_last;
  __shared__ float2 s_top[kMostWindow];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int b = static_cast<int>(blockIdx.x) / p.cluster, rank = static_cast<int>(blockIdx.x) - b * p.cluster;
  pdl_launch_dependents();
  pdl_wait();
  const int lo = p.cu ? p.cu[b] : b, hi = p.cu ? p.cu[b + 1] : b + 1;
  const int start = min(max(lo, 0), p.num_tokens);
  const int n = min(max(min(hi, p.num_tokens) - start, 0), p.max_seqlen);
  long long* const out_tokens = p.out_tokens + static_cast<long long>(b) * p.max_seqlen;
  int* const out_rows = p.out_rows + static_cast<long long>(b) * p.max_seqlen;
  if (n == 0) {  // the whole cluster
    if (rank == 0) {
      for (int i = tid; i < p.max_seqlen; i += kVerifyThreads) {
        out_tokens[i] = -1;
        out_rows[i] = -1;
      }
      if (tid == 0) p.out_counts[b] = 0;
    }
    return;
  }
  // (none writes to another block's shared memory before that has started: the wait for this comes ahead of the first exchange)
  if (p.cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const T* const logits = static_cast<const T*>(p.logits) + static_cast<long long>(start) * p.logits_stride;
  const float* const probs = p.probs ? p.probs + static_cast<long long>(start) * p.probs_stride : nullptr;
  const bool chain = p.parents == nullptr;
  const int my_warp = rank * kVerifyWarps + warp;
  auto row_at = [&](int r) { return Row<T>(logits + r * p.logits_stride, p.vocab); };
  auto begin_of_block = [&](const Row<T>& row, int r) { return min(row.words, p.per_block * r); };
  // a warp's words of a row, where each row is shared out over the warps
  auto begin_of = [&](const Row<T>& row, int w) { return min(row.words, p.per_warp * w); };
  auto first_child = [&](int r) { return chain ? r + 1 : s_first[r]; };  // n or more: none
  auto meet = [&] { meet_of(p.cluster); };

  const uint32_t ring = smem_u32(s_ring) + (warp * (kDepth * 32) + lane) * 16;  // a lane's words lie 512 bytes apart

  // ---- the rows: their parents, tokens, and what their parents' logits and the draft say of them (these are taken to shared memory when they are needed) ----
  const float heat = p.temperatures ? p.temperatures[b] : 1.f;
  float my_x = -CUDART_INF_F, my_q = 0.f;
  if (tid < n) {
    const int up = chain ? tid - 1 : tid > 0 ? p.parents[start + tid] : -1;
    const long long token = p.tokens ? p.tokens[start + tid] : -1;
    const bool child = up >= 0 && up < tid && token >= 0 && token < p.vocab;  // (a token outside the vocabulary is never taken)
    s_parent[tid] = up >= 0 && up < tid ? up : -1;
    s_token[tid] = child ? static_cast<int>(token) : -1;
    s_first[tid] = kMostDrafted;
    s_coin[tid] = p.coins ? p.coins[start + tid] : 0.f;
    if (child) {
      my_x = number(logits[up * p.logits_stride + token]);
      if (probs) my_q = probs[up * p.probs_stride + token];
    }
  }
  if (tid >= kVerifyThreads - kSteps) {
    const int i = tid - (kVerifyThreads - kSteps);
    s_power[i] = exp2(i * (1.0 / kSteps));
  }
  __syncthreads();
  if (!chain) {
    if (tid < n && s_parent[tid] >= 0) atomicMin(&s_first[s_parent[tid]], tid);
    __syncthreads();
  }
  const bool greedy = !(heat > 0.f);
  const double inverse = greedy ? 1.0 : 1.0 / static_cast<double>(heat);
  const float per_unit = fminf(static_cast<float>(inverse * 1.4426950408889634), 3.0e38f);  // in octaves
  int turn = 0, turn_sum = 0;  // of the cluster's exchanges: their places alternate, so that none is written while a block still reads the one before
  Weigh weigh{inverse * (kSteps * 1.4426950408889634), 16384.0 / (inverse * (kSteps * 1.4426950408889634)), 0.0, smem_u32(s_power), 0.f, false};

  int node = 0, accepted = 0;
  bool met = p.cluster == 1;
  float top = 0.f;     // of the current row
  double total = 0.0;  //   its sum, of 32 bits or of 64
  // sums over the cluster's warps: their shares stay in s_share, the blocks' in s_shares of the turn before
  auto share_out = [&](const Shares& mine_of) {
    double v[3] = {mine_of.all, mine_of.drawn, mine_of.draft};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], m);
      if (lane == 0) s_share[i][warp] = v[i];
    }
    __syncthreads();
    if (warp < 3) {
      double mine = lane < kVerifyWarps ? s_share[warp][lane] : 0.0;
#pragma unroll
      for (int m = 16; m >= 1; m >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, m);
      if (p.cluster == 1) s_shares[turn_sum][warp][0] = mine;
      else if (lane < p.cluster) put_peer(&s_shares[turn_sum][warp][rank], lane, mine);
    }
    meet();
    turn_sum ^= 1;
  };
  auto shares_of_row = [&](int r, const float* q, int num_kids) {
    const Row<T> row = row_at(r);
    const int w0 = begin_of(row, my_warp), w1 = begin_of(row, my_warp + 1);
    if (weigh.odd) {
      return q ? shares_of<T, true, true>(row.p, p.vocab, w0, w1, q, total, weigh, nullptr, 0)
               : shares_of<T, false, true>(row.p, p.vocab, w0, w1, nullptr, 0.0, weigh, s_kids, num_kids);
    }
    return q ? shares_of<T, true, false>(row.p, p.vocab, w0, w1, q, total, weigh, nullptr, 0)
             : shares_of<T, false, false>(row.p, p.vocab, w0, w1, nullptr, 0.0, weigh, s_kids, num_kids);
  };
  auto sum_of = [&](int i) {
    double sum = 0.0;
    for (int r = 0; r < p.cluster; ++r) sum += s_shares[turn_sum ^ 1][i][r];
    return sum;
  };
  // A warp's decision on row r with largest number m (or, greedy, largest token) and sum of weights: the child that is taken, 0 for none, -1 where this could err.  In
  // Real's bits.  With those of 32 the two sides are off by no more than 2 (doubt + 1e-7 times the child's octaves below m) of themselves: a weight's exponent is off by
  // 3 2^-24 of itself, ln(2) of which it makes of the weight, 1.24e-7 an octave; and by 1e-37 where numbers are next to 32 bits' smallest.
  auto decide = [&](int r, float m, auto sum, int largest, auto doubt) {
    using Real = decltype(sum);
    constexpr bool kFast = sizeof(Real) == 4;
    if (kFast && !greedy && !(sum >= Real(0.5) && sum < Real(1e30))) return -1;
    const Real u = static_cast<Real>(s_coin[r]);
    Real mass = 0;
    for (int i0 = (r + 1) & ~31; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      const bool child = i < n && i > r && s_parent[i] == r && s_token[i] >= 0;
      if (!__any_sync(0xffffffffu, child)) continue;
      bool take = child && s_token[i] == largest, close = false;
      if (!greedy) {
        Real w = 0, down = 0;
        if (child && !s_again[i]) {
          if constexpr (kFast) {
            down = (s_x[i] - m) * per_unit;
            w = ex2(down);
          } else {
            w = weigh(s_x[i]);
          }
        }
        Real left = u * sum, right = w;
        if (probs) {
          left *= static_cast<Real>(child ? s_q[i] : 0.f);
        } else {
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const Real below = __shfl_up_sync(0xffffffffu, right, d);
            if (lane >= d) right += below;
          }
          right += mass;
          mass = __shfl_sync(0xffffffffu, right, 31);
        }
        take = child && w > Real(0) && left < right;
        if constexpr (kFast) close = child && !(fabsf(left - right) > (doubt - 1e-7f * fmaxf(down, -150.f)) * (left + right) + 1e-37f);  // (150 octaves: nothing)
      }
      const unsigned first = __ballot_sync(0xffffffffu, take), border = __ballot_sync(0xffffffffu, close);
      if (border && (!first || __ffs(border) <= __ffs(first))) return -1;  // (one behind the first that is taken decides nothing)
      if (first) return i0 + __ffs(first) - 1;
    }
    return 0;
  };
  // a warp's lanes hold parts of a row's maximum and sum, or word: joined in all of them
  auto join = [&](float& m, float& s, int& word) {
    float most = m;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    if (greedy) {
      if (m != most) word = 0x7fffffff;
      word = __reduce_min_sync(0xffffffffu, word);
    } else {
      s *= ex2((m - fmaxf(most, -3.4028235e38f)) * per_unit);
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    }
    m = most;
  };

  if (tid == 0) s_path[0] = 0;
  for (bool walking = true; walking;) {
    // ---- maxima and sums of the window's rows: the block's words of all of them one behind the other, shared out over the warps in groups of 128 ----
    int count = 0;
    for (int r = node; r < n && count < p.window; r = first_child(r)) ++count;
    // of a row that the warp has no share of; or whose words lie within it
    if (lane < count) s_part[lane][warp] = make_uint2(0xff800000u, greedy ? 0x7fffffffu : 0u);
    if (warp < count && lane == 0) s_part[warp][kVerifyWarps] = make_uint2(0xff800000u, greedy ? 0x7fffffffu : 0u);
    __syncwarp();
    // (of a row where words begin at another of its numbers than in the next, a group may be empty)
    const int per_row = (p.per_block + 32 * kGroup - 1) / (32 * kGroup), groups = count * per_row;
    const int group0 = groups * warp / kVerifyWarps, group1 = groups * (warp + 1) / kVerifyWarps;
    struct Place {
      int k, in_row, word, end;  // row of the window, group of the row; this lane's first word of the group and the end of the block's
      const uint4* from;
    };
    auto open = [&](Place& at) {
      int r = node;
      for (int k = 0; k < at.k; ++k) r = first_child(r);
      const Row<T> row = row_at(r);
      const int w0 = begin_of_block(row, rank), w1 = begin_of_block(row, rank + 1), b0 = row.whole_from(w0, w1);
      at.word = b0 + at.in_row * (32 * kGroup) + lane;
      at.end = row.whole_to(b0, w1);
      at.from = row.at(at.word);
    };
    auto forth = [&](Place& at) {
      if (++at.in_row == per_row) {
        at.in_row = 0;
        if (++at.k < count) open(at);
      } else {
        at.word += 32 * kGroup;
        at.from += 32 * kGroup;
      }
    };
    Place here{group0 / per_row, group0 % per_row, 0, 0, nullptr};
    if (group0 < group1) open(here);
    Place there = here;
    int copied = group0;
    auto copy_group = [&] {
      if (copied < group1) {
        const uint32_t to = ring + (copied & (kStages - 1)) * (kGroup * 512);
        if (there.word - lane + 32 * kGroup <= there.end) {
#pragma unroll
          for (int e = 0; e < kGroup; ++e) copy16(to + e * 512, there.from + 32 * e);
        } else {
#pragma unroll 1
          for (int e = 0; e < kGroup; ++e)
            if (there.word + 32 * e < there.end) copy16(to + e * 512, there.from + 32 * e);
        }
        forth(there);
        ++copied;
      }
      copies_commit();
    };
    for (int i = 0; i < kStages - 1; ++i) copy_group();
    float m = -CUDART_INF_F, s = 0.f;
    int word = 0x7fffffff;
    // one word more of a lane, or several: `words` at most
    auto take = [&](const uint4 (&its)[kGroup], int words, int at_word) {
      float most[kGroup], largest = -CUDART_INF_F;
#pragma unroll
      for (int e = 0; e < kGroup; ++e) {
        most[e] = largest_of<T>(its[e]);
        largest = fmaxf(largest, most[e]);
      }
      if (greedy) {
        int lowest = 0x7fffffff;
#pragma unroll
        for (int e = kGroup - 1; e >= 0; --e)
          if (e < words && most[e] == largest) lowest = at_word + 32 * e;
        word = largest > m ? lowest : largest == m ? min(word, lowest) : word;
        m = fmaxf(m, largest);
        return;
      }
      // (a product and a difference in one rounding: off by 2^-24 of top / t, which the doubt below counts)
      const float m_new = fmaxf(m, largest), ref = m_new == -CUDART_INF_F ? 0.f : m_new, off = -ref * per_unit;
      const f2 k2 = pack2(per_unit, per_unit), off2 = pack2(off, off);
      f2 sum[2] = {pack2(s * ex2((m - ref) * per_unit), 0.f), pack2(0.f, 0.f)};
      m = m_new;
#pragma unroll
      for (int e = 0; e < kGroup; ++e) {
        if (e >= words) break;  // (all lanes alike)
        float x[kN];
        numbers_of<T>(its[e], x);
#pragma unroll
        for (int i = 0; i < kN; i += 2) {
          const float2 y = unpack2(fma2(pack2(x[i], x[i + 1]), k2, off2));
          sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pack2(ex2(y.x), ex2(y.y)));
        }
      }
      const float2 both = unpack2(add2(sum[0], sum[1]));
      s = both.x + both.y;
    };
    constexpr uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;  // -inf
    // The words that reach past a row, of row k by warp k ahead of its groups: with them as its share of the row if the groups are of another one
    for (int g = group0 - (warp < count ? 1 : 0); g < group1; ++g) {
      uint4 its[kGroup];
      auto none = [&] {
#pragma unroll
        for (int e = 0; e < kGroup; ++e) its[e] = make_uint4(kNone, kNone, kNone, kNone);
      };
      int words = 1, at_word = 0, of = warp;
      bool ends = true;
      if (g < group0) {
        int r = node;
        for (int k = 0; k < warp; ++k) r = first_child(r);
        const Row<T> row = row_at(r);
        const int w0 = begin_of_block(row, rank), w1 = begin_of_block(row, rank + 1), b0 = row.whole_from(w0, w1), b1 = row.whole_to(b0, w1);
        if (b0 == w0 && b1 == w1) continue;  // (all lanes alike)
        at_word = lane == 0 ? w0 : w1 - 1;
        none();
        if (lane == 0 ? b0 > w0 : lane == 1 && b1 < w1) its[0] = row.word(at_word);
      } else {
        copy_group();
        copies_wait<kStages - 1>();
        const uint32_t from = ring + (g & (kStages - 1)) * (kGroup * 512);
        if (here.word - lane + 32 * kGroup <= here.end) {
#pragma unroll
          for (int e = 0; e < kGroup; ++e) its[e] = take16(from + e * 512);
        } else {
          none();
#pragma unroll
          for (int e = 0; e < kGroup; ++e)
            if (here.word + 32 * e < here.end) its[e] = take16(from + e * 512);
        }
        words = (here.end - here.word + lane + 31) >> 5;
        at_word = here.word;
        of = here.k;
        ends = here.in_row + 1 == per_row || g + 1 == group1;
        forth(here);
      }
      take(its, words, at_word);
      if (!ends) continue;
      join(m, s, word);
      if (lane == 0) s_part[of][g < group0 ? kVerifyWarps : warp] = make_uint2(__float_as_uint(m), greedy ? static_cast<uint32_t>(word) : __float_as_uint(s));
      m = -CUDART_INF_F;
      s = 0.f;
      word = 0x7fffffff;
    }
    copies_wait<0>();
    if (node == 0 && tid < n) {
      s_x[tid] = my_x;
      s_q[tid] = my_q;
      bool again = false;
      if (!chain && s_token[tid] >= 0)
        for (int j = s_parent[tid] + 1; j < tid; ++j) again |= s_parent[j] == s_parent[tid] && s_token[j] == s_token[tid];
      s_again[tid] = again;
    }
    __syncthreads();
    if (!met) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    met = true;
    auto parts_of = [&](const uint2* parts, int many, float& m, float& s, int& word) {
      const uint2 mine = lane < many ? parts[lane] : make_uint2(0xff800000u, 0u);
      m = __uint_as_float(mine.x);
      s = __uint_as_float(mine.y);
      word = lane < many ? static_cast<int>(mine.y) : 0x7fffffff;
      join(m, s, word);
    };
    if (warp < count) {
      float m, s;
      int word;
      parts_of(s_part[warp], kVerifyWarps + 1, m, s, word);
      const uint2 both = make_uint2(__float_as_uint(m), greedy ? static_cast<uint32_t>(word) : __float_as_uint(s));
      if (p.cluster == 1) s_all[turn][warp][0] = both;
      else if (lane < p.cluster) put_peer(&s_all[turn][warp][rank], lane, both);
    }
    meet();
    // ---- a warp decides a row ----
    if (warp < count) {
      int r = node, word, largest = -1;
      for (int k = 0; k < warp; ++k) r = first_child(r);
      float m, s;
      parts_of(s_all[turn][warp], p.cluster, m, s, word);
      if (greedy && m > -CUDART_INF_F) {
        const Row<T> row = row_at(r);
        const uint4 its = row.word(word);
        const T* x = reinterpret_cast<const T*>(&its);
#pragma unroll
        for (int i = kN - 1; i >= 0; --i)
          if (number(x[i]) == m) largest = word * kN - row.skip + i;
      }
      // A weight of 32 bits is off by 2^-24 of the numbers that its exponent comes from, top / t and their difference of 40 octaves (what is less says nothing in the
      // sum), and by ex2's 2^-22; the sum by 2^-24 for each number that a lane adds to what it has: in every group a fourth of its numbers, those of its own two halves,
      // and five for the scaling where the maximum moves.  (Equal weights are all rounded one way: 2^20 of them beside a larger one, in a block, 4.8e-5.)
      const int serial = (min(per_row, (groups + kVerifyWarps - 1) / kVerifyWarps) + 2) * (kGroup * kN / 4 + 8);
      const int taken = decide(r, m, s, largest, 1e-5f + fabsf(m * per_unit) * 2.4e-7f + static_cast<float>(serial) * 2.9802322e-8f);
      if (lane == 0) {
        s_next[warp] = taken;
        s_largest[warp] = largest;
        s_top[warp] = make_float2(m, s);
      }
    }
    __syncthreads();
    // ---- the walk, all threads of the cluster alike ----
    for (int k = 0; k < count; ++k) {
      int taken = s_next[k];
      top = s_top[k].x;
      total = s_top[k].y;
      if (taken < 0) {
        weigh.against(top);
        share_out(shares_of_row(node, nullptr, 0));
        total = sum_of(0);
        if (warp == 0) {
          const int t = decide(node, top, total, -1, 0.0);
          if (lane == 0) s_next[k] = t;
        }
        __syncthreads();
        taken = s_next[k];
      }
      if (greedy && tid == 0) s_last = s_largest[k];
      if (taken == 0) {  // the row that the sequence ends with
        walking = false;
        break;
      }
      const bool inside = taken == first_child(node);
      node = taken;
      ++accepted;
      if (tid == 0) s_path[accepted] = node;
      if (!inside) break;
    }
    turn ^= 1;
    __syncthreads();  // s_next, s_part
  }

  // ---- the token behind the last accepted row ----
  if (!greedy && top == -CUDART_INF_F) {
    if (tid == 0) s_last = -1;
  } else if (!greedy) {
    weigh.against(top);
    const Row<T> row = row_at(node);
    const bool rejected = first_child(node) < n;
    const float* const q = rejected && probs ? probs + node * p.probs_stride : nullptr;
    if (warp == 0) {
      int many = 0;
      for (int i0 = 0; rejected && !probs && i0 < n; i0 += 32) {
        const int i = i0 + lane;
        const bool kid = i < n && s_parent[i] == node && s_token[i] >= 0;
        const unsigned kids = __ballot_sync(0xffffffffu, kid);
        if (kid) s_kids[many + __popc(kids & ((1u << lane) - 1))] = s_token[i];
        many += __popc(kids);
      }
      if (lane == 0) s_num_kids = many;
    }
    __syncthreads();
    auto kids_in = [&](int w0, int w1) {  // how many of them there are to look for in these words
      bool any = false;
      for (int j = 0; j < s_num_kids; ++j) any |= s_kids[j] >= w0 * kN - row.skip && s_kids[j] < w1 * kN - row.skip;
      return any ? s_num_kids : 0;
    };
    // With e the weights, S their sum and s that sum as 32 bits have it: what is drawn from is max(e - S q, 0).  S is not known before the row's end; but
    // sum (e - S q) over a run is sum (e - s q) + (s - S) sum q, over the numbers above zero: one pass.  Those for which e / q lies between s and S are counted
    // on the wrong side by it, so what is drawn from is off by |s - S| times their share of q.  Where that may be more than 1e-4 of all of it -- a draft next to the
    // target, down to one that is the target's best token, of which S q takes all that s q leaves -- the token is drawn number by number.
    share_out(shares_of_row(node, q, kids_in(begin_of(row, my_warp), begin_of(row, my_warp + 1))));
    const double all = sum_of(0), correction = total - all;
    const double (&shares)[3][kMostBlocks] = s_shares[turn_sum ^ 1];
    double whole = 0.0;
    for (int r = 0; r < p.cluster; ++r) whole += fmax(q ? shares[1][r] + correction * shares[2][r] : shares[1][r], 0.0);
    const bool exactly = q && correction != 0.0 && !(whole >= 1e4 * fabs(correction));  // the cluster's threads all alike
    if (exactly) draw_exactly<T>(row.p, p.vocab, q, all, weigh, p.draws[b], s_share[0], s_shares[turn_sum][0], s_shares[turn_sum][1], p.cluster, rank, out_tokens + accepted);
    const bool from_p = !(whole > kNothing);  // nothing is left of what was asked for
    if (from_p) whole = all;
    // Which of up to 16 shares the threshold falls into, given what lies ahead of them (then: of the one chosen); the last with any where it falls behind them all
    const double threshold = static_cast<double>(p.draws[b]) * whole;
    auto choose = [&](double mine, double run, double& ahead) {  // run: of the shares up to this one
      const unsigned any = __ballot_sync(0xffffffffu, mine > kNothing), past = __ballot_sync(0xffffffffu, mine > kNothing && ahead + run > threshold);
      const int chosen = past ? __ffs(past) - 1 : 31 - __clz(any);
      ahead += __shfl_sync(0xffffffffu, run - mine, chosen & 31);
      return chosen;
    };
    auto run_of = [&](double x) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double below = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += below;
      }
      return x;
    };
    auto runs_of = [&](double& x, double& y) {  // (both at once: a step is a shuffle's and a sum's latency)
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double below_x = __shfl_up_sync(0xffffffffu, x, d), below_y = __shfl_up_sync(0xffffffffu, y, d);
        if (lane >= d) {
          x += below_x;
          y += below_y;
        }
      }
    };
    auto share_of = [&](const double* of_all, const double* of_drawn, const double* of_draft, int many) {
      if (lane >= many) return 0.0;
      return from_p ? of_all[lane] : fmax(q ? of_drawn[lane] + correction * of_draft[lane] : of_drawn[lane], 0.0);
    };
    double ahead = 0.0;
    const double of_block = share_of(shares[0], shares[1], shares[2], p.cluster), of_mine = share_of(s_share[0], s_share[1], s_share[2], kVerifyWarps);
    double run_block = of_block, run_mine = of_mine;
    runs_of(run_block, run_mine);
    if (!exactly && choose(of_block, run_block, ahead) == rank) {
      // the warp, then its run shared out over all of the block's lanes, then the number
      const int of = rank * kVerifyWarps + choose(of_mine, run_mine, ahead);
      const int w0 = begin_of(row, of), len = begin_of(row, of + 1) - w0;
      const int c0 = w0 + static_cast<int>(static_cast<long long>(len) * tid / kVerifyThreads), c1 = w0 + static_cast<int>(static_cast<long long>(len) * (tid + 1) / kVerifyThreads);
      const int kids = !q && !from_p ? kids_in(w0, w0 + len) : 0;
      const float floor = top == CUDART_INF_F ? 3.4028235e38f : weigh.least;
      double w[kN], sum = 0.0;  // of a word's numbers the sums up to them, from the lane's first on
      unsigned some = 0;        // those with a weight
      auto sums_of = [&](int c) {
        const int first = c * kN - row.skip;
        float x[kN], qs[kN];  // (all of q's on their way with the word)
#pragma unroll
        for (int k = 0; k < kN; ++k) qs[k] = q && static_cast<unsigned>(first + k) < static_cast<unsigned>(p.vocab) ? __ldcg(q + first + k) : 0.f;
        numbers_of<T>(row.word(c), x);
#pragma unroll
        for (int k = 0; k < kN; ++k) w[k] = x[k] > floor ? (top == CUDART_INF_F ? 1.0 : weigh.finite(x[k])) : 0.0;
        for (int j = 0; j < kids; ++j) {
          const int at = s_kids[j] - first;
#pragma unroll
          for (int k = 0; k < kN; ++k)
            if (k == at) w[k] = 0.0;
        }
        some = 0;
#pragma unroll
        for (int k = 0; k < kN; ++k) {
          if (q && !from_p) w[k] = w[k] > 0.0 ? fmax(fma(-all, static_cast<double>(qs[k]), w[k]), 0.0) : 0.0;
          some |= w[k] > 0.0 ? 1u << k : 0u;
          w[k] = sum += w[k];
        }
      };
      // (The code of this is run through for the first time here and waits for its instructions, so it is there once: for the sums, and, for the chosen lane's numbers
      // if it has several words, again.)
      const int words = (len + kVerifyThreads - 1) / kVerifyThreads;  // of a lane at most
      int i = 0, found = -1, last = -1;                               // the first past the threshold; the last with any weight
      bool chosen = false;
#pragma unroll 1
      while (true) {
        if (c0 + i < c1) sums_of(c0 + i);
        if (!chosen) {
          if (++i < words) continue;
          const double run = run_of(sum);
          __syncthreads();  // s_share has been read
          if (lane == 31) s_share[0][warp] = run;
          __syncthreads();
          const double of_warp = lane < kVerifyWarps ? s_share[0][lane] : 0.0;
          const int in = choose(of_warp, run_of(of_warp), ahead);
          if (in < 0) {  // the share was rounding of sum q's 32 bits, none of its numbers is above zero: this block draws by itself
            draw_exactly<T>(row.p, p.vocab, from_p ? nullptr : q, all, weigh, p.draws[b], s_share[0], s_shares[turn_sum][0], s_shares[turn_sum][1], 1, 0, out_tokens + accepted);
            break;
          }
          if (in != warp || choose(sum, run, ahead) != lane) break;
          chosen = true;
          i = 0;
          if (words > 1) {
            sum = 0.0;
            continue;
          }
        }
#pragma unroll
        for (int k = kN - 1; k >= 0; --k) {
          if (!(some >> k & 1u)) continue;
          const int token = (c0 + i) * kN - row.skip + k;
          if (ahead + w[k] > threshold) found = token;
          last = max(last, token);
        }
        if (found >= 0 || c0 + ++i >= c1) {
          out_tokens[accepted] = found >= 0 ? found : last;
          break;
        }
      }
    }
  }
  __syncthreads();
  if (rank == 0) {
    for (int i = tid; i < p.max_seqlen; i += kVerifyThreads) {
      out_rows[i] = i <= accepted ? s_path[i] : -1;
      if (i != accepted) out_tokens[i] = i < accepted ? s_token[s_path[i + 1]] : -1;
      else if (greedy || top == -CUDART_INF_F) out_tokens[i] = s_last;
    }
    if (tid == 0) p.out_counts[b] = accepted + 1;
  }
}

template <typename T>
int launch_verify(VerifyParams p, int batch, void* stream) {
  static std::atomic<bool> done[kMaxDevices] = {};  // of this type
  std::atomic<bool>& d = done[device_ordinal()];
  if (!d.load(std::memory_order_relaxed)) {
    const int rc = check_cuda(cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes), "verify_drafts: shared memory");
    if (rc) return rc;
    const int rn = check_cuda(cudaFuncSetAttribute(verify_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1), "verify_drafts: clusters of sixteen");
    if (rn) return rn;
    d.store(true, std::memory_order_relaxed);
  }
  // Blocks of a sequence: as many as find places for all sequences at once.  (Of sixteen, eight and four blocks 7, 15 and 32 clusters do, where 148 / 16 is 9.  Sequences
  // that wait for the first ones' places, and fewer blocks, of powers of two: 8 chains of 5, 128256 tokens, 31.0 us and 21.4; 16 of them 36.5 and 28.9; 36 47.4 and 41.2.
  // Of any number, without probabilities: 19.2, 22.5 and 31.2.)
  static std::atomic<int> held[kMaxDevices][kMostBlocks + 1] = {};
  auto places = [&](int n) { return paged::clusters_at_once(held[device_ordinal()][n], verify_kernel<T>, kVerifyThreads, kRingBytes, n); };
  p.cluster = paged::most_blocks_at_once(places, kMostBlocks, batch);
  const long long words = (static_cast<long long>(p.vocab) + 2 * Row<T>::kN - 2) / Row<T>::kN;  // of a row that begins at a word's last number
  auto share = [&](int of) { return static_cast<int>((words + 32ll * of - 1) / (32ll * of) * 32); };  // (a warp takes 32 at a time in any case)
  p.per_block = share(p.cluster);
  p.per_warp = share(p.cluster * kVerifyWarps);
  return paged::launch(verify_kernel<T>, dim3(static_cast<unsigned>(batch) * p.cluster), kVerifyThreads, kRingBytes, stream, "verify_drafts", p.cluster, p);
}

}  // namespace

int draft_tree(int* positions, long long* visible, const int* parents, const int* cu, const int* lengths, int batch, int num_tokens, int max_seqlen, void* stream) {
  if (batch == 0 || num_tokens == 0 || max_seqlen == 0) return QS_OK;
  const int threads = (max_seqlen + 31) / 32 * 32, words = (max_seqlen + 63) / 64;
  return paged::launch(tree_kernel, dim3(batch), threads, 0, stream, "draft_tree", 1, positions, reinterpret_cast<unsigned long long*>(visible), parents, cu, lengths, num_tokens,
                       max_seqlen, words);
}

int verify_drafts(const VerifyArgs& a) {
  if (a.batch == 0) return QS_OK;
  VerifyParams p{};
  p.logits = a.logits; p.logits_stride = a.logits_stride; p.probs_stride = a.probs_stride; p.tokens = a.tokens; p.parents = a.parents; p.probs = a.probs; p.cu = a.cu_seqlens;
  p.coins = a.coins; p.draws = a.draws; p.temperatures = a.temperatures; p.out_tokens = a.out_tokens; p.out_rows = a.out_rows; p.out_counts = a.out_counts;
  p.num_tokens = a.num_tokens; p.vocab = a.vocab; p.max_seqlen = a.max_seqlen;
  // Rows of a window: of a chain all, for the slowest sequence of a batch is likely to walk it to the end (64 chains of 6, 128256 tokens: a row at a time 59 us); of a
  // tree, where the first child is one of several, few
  p.window = a.parents ? 2 : kMostWindow;
  return a.type == 0 ? launch_verify<__half>(p, a.batch, a.stream) : a.type == 1 ? launch_verify<__nv_bfloat16>(p, a.batch, a.stream) : launch_verify<float>(p, a.batch, a.stream);
}

}  // namespace qs
