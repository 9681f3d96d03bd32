// qserve_b200 -- drafted tokens of a step: what the rows of a tree see of one another, and their verification against the target's probabilities.
//
// The rows of sequence b are a portion (as in paged_cache.cu): row 0 the token that the step starts from, every other one a drafted token with a parent
// among the rows ahead of it.  Row i's logits are the target's behind row i, so they judge i's children.
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
// tree: thread = row, up the ancestors
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
// ------------------------------------------------------------------------------------------------------------------------
constexpr int kVerifyWarps = 16, kVerifyThreads = 32 * kVerifyWarps, kMostBlocks = 8;
constexpr int kWindow = 8;  // rows whose maxima and sums are taken together at most
static_assert(kVerifyThreads >= kMostDrafted, "a thread per row");

template <typename T>
struct Chunk {
  static constexpr int kN = 16 / sizeof(T);
};
template <typename T>
__device__ __forceinline__ float number(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __half2float(x);
  else return __bfloat162float(x);
}

// A row of logits in 16-byte words: word c holds the numbers kN c - skip .. + kN - 1
template <typename T>
struct Row {
  const T* p;
  int skip, vocab, words;
  __device__ __forceinline__ Row(const T* row, int v) : p(row), vocab(v) {
    skip = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    words = (skip + v + Chunk<T>::kN - 1) / Chunk<T>::kN;
  }
  // numbers that are none, and those outside the row: -inf
  __device__ __forceinline__ uint4 raw(int c) const {
    constexpr int kN = Chunk<T>::kN;
    const int first = c * kN - skip;
    if (first >= 0 && first + kN <= vocab) return __ldg(reinterpret_cast<const uint4*>(p + first));
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
  int num_tokens, vocab, max_seqlen, cluster, log2_warps;  // of the cluster
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void put_peer(const double* mine, uint32_t rank, double v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(a), "d"(v) : "memory");
}
__device__ __forceinline__ void put_peer(const uint2* mine, uint32_t rank, uint2 v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(mine)), "r"(rank));
  asm volatile("st.shared::cluster.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(v.x), "r"(v.y) : "memory");
}

// What a number weighs against its row's largest one, in 64 bits: exp((x - top) / t); where the largest has no end, those without one alone
__device__ __forceinline__ double weight(float x, float top, double per_unit) {
  if (x == top) return 1.0;
  if (!(x < top) || x == -CUDART_INF_F || top == CUDART_INF_F) return 0.0;  // no number, none left, no end
  return exp((static_cast<double>(x) - static_cast<double>(top)) * per_unit);
}

template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const __grid_constant__ VerifyParams p) {
  constexpr int kN = Chunk<T>::kN;
  __shared__ int s_parent[kMostDrafted], s_token[kMostDrafted], s_first[kMostDrafted], s_path[kMostDrafted];
  __shared__ int s_kids[kMostDrafted];                        // tokens of the last row's children
  __shared__ float s_x[kMostDrafted], s_q[kMostDrafted], s_coin[kMostDrafted];
  __shared__ unsigned char s_again[kMostDrafted];
  __shared__ uint2 s_part[kWindow][kVerifyWarps];             // of a warp: maximum, and sum or word
  __shared__ uint2 s_all[2][kWindow][kMostBlocks];            // of the cluster's blocks
  __shared__ double s_sum[kVerifyWarps], s_sums[2][kMostBlocks];
  __shared__ int s_next, s_last, s_num_kids;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int rank = static_cast<int>(blockIdx.x) % p.cluster, b = static_cast<int>(blockIdx.x) / p.cluster;
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
  const float heat = p.temperatures ? p.temperatures[b] : 1.f;
  const bool greedy = !(heat > 0.f);
  const double per_unit = greedy ? 1.0 : 1.0 / static_cast<double>(heat);
  const float per_unit_log2 = fminf(static_cast<float>(per_unit * 1.4426950408889634), 3.0e38f);
  const T* const logits = static_cast<const T*>(p.logits) + static_cast<long long>(start) * p.logits_stride;
  const float* const probs = p.probs ? p.probs + static_cast<long long>(start) * p.probs_stride : nullptr;

  // ---- the rows: their parents, tokens, and what their parents' logits and the draft say of them ----
  if (tid < n) {
    const int up = p.parents ? (tid > 0 ? p.parents[start + tid] : -1) : tid - 1;
    const long long token = p.tokens ? p.tokens[start + tid] : -1;
    const bool child = up >= 0 && up < tid && token >= 0 && token < p.vocab;  // (a token outside the vocabulary is never taken)
    s_parent[tid] = up >= 0 && up < tid ? up : -1;
    s_token[tid] = child ? static_cast<int>(token) : -1;
    s_x[tid] = child ? number(logits[up * p.logits_stride + token]) : -CUDART_INF_F;
    s_q[tid] = child && probs ? probs[up * p.probs_stride + token] : 0.f;
    s_coin[tid] = p.coins ? p.coins[start + tid] : 0.f;
    s_first[tid] = kMostDrafted;
  }
  __syncthreads();
  if (tid < n) {
    const int up = s_parent[tid], token = s_token[tid];
    if (up >= 0) atomicMin(&s_first[up], tid);
    bool again = false;
    if (p.parents && token >= 0)
      for (int j = 1; j < tid; ++j) again |= s_parent[j] == up && s_token[j] == token;
    s_again[tid] = again;
  }
  __syncthreads();

  const int my_warp = rank * kVerifyWarps + warp;
  int turn = 0, turn_sum = 0;  // of the cluster's exchanges: their places alternate, so that none is written while a block still reads the one before
  // a warp's words of a row
  auto begin_of = [&](const Row<T>& row, int w) { return static_cast<int>((static_cast<long long>(row.words) * w) >> p.log2_warps); };

  // sums of 64 bits over the cluster, the same in all of its threads: the warps' shares stay in s_sum, the blocks' in s_sums
  auto cluster_sum = [&](double v) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if (lane == 0) s_sum[warp] = v;
    __syncthreads();
    if (warp == 0) {
      double mine = 0.0;
      for (int w = 0; w < kVerifyWarps; ++w) mine += s_sum[w];
      if (lane < p.cluster) put_peer(&s_sums[turn_sum][rank], lane, mine);
    }
    cluster_sync();
    double all = 0.0;
    for (int r = 0; r < p.cluster; ++r) all += s_sums[turn_sum][r];
    turn_sum ^= 1;
    return all;
  };
  // f(index of the first number, the word's numbers) over this warp's words of a row
  auto over = [&](const Row<T>& row, int w0, int w1, auto f) {
    for (int c0 = w0; c0 < w1; c0 += 64) {
      uint4 raw[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (c0 + 32 * k + lane < w1) raw[k] = row.raw(c0 + 32 * k + lane);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (c0 + 32 * k + lane < w1) f((c0 + 32 * k + lane) * kN - row.skip, reinterpret_cast<const T*>(&raw[k]));
    }
  };
  auto exact_sum = [&](int row_of, float top) {
    const Row<T> row(logits + row_of * p.logits_stride, p.vocab);
    double sum = 0.0;
    over(row, begin_of(row, my_warp), begin_of(row, my_warp + 1), [&](int, const T* x) {
#pragma unroll
      for (int k = 0; k < kN; ++k) sum += weight(number(x[k]), top, per_unit);
    });
    return cluster_sum(sum);
  };

  int node = 0, accepted = 0;
  if (tid == 0) s_path[0] = 0;
  float top = 0.f;      // of the current row
  int best_word = 0;    //   greedy: the word of its largest number
  for (bool walking = true; walking;) {
    // ---- maxima and sums of the rows of a window: the current one and those behind it if every first child is taken ----
    int count = 0;
    for (int at = node; count < kWindow && at < n; at = s_first[at], ++count) {
      const Row<T> row(logits + at * p.logits_stride, p.vocab);
      const int w0 = begin_of(row, my_warp), w1 = begin_of(row, my_warp + 1);
      float m = -CUDART_INF_F, s = 0.f;
      int word = 0x7fffffff;
      for (int c0 = w0; c0 < w1; c0 += 128) {
        uint4 raw[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c0 + 32 * e + lane < w1) raw[e] = row.raw(c0 + 32 * e + lane);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (c0 + 32 * e + lane >= w1) break;
          const T* x = reinterpret_cast<const T*>(&raw[e]);
          float v[kN], most = -CUDART_INF_F;
#pragma unroll
          for (int i = 0; i < kN; ++i) {
            v[i] = number(x[i]);
            most = fmaxf(most, v[i]);  // (passes over what is no number)
          }
          if (greedy) {
            if (most > m) word = c0 + 32 * e + lane;
            m = fmaxf(m, most);
          } else {
            const float m_new = fmaxf(m, most), ref = fmaxf(m_new, -3.4028235e38f);
            s *= ex2((m - ref) * per_unit_log2);
#pragma unroll
            for (int i = 0; i < kN; ++i) s += ex2((v[i] - ref) * per_unit_log2);
            m = m_new;
          }
        }
      }
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, d), os = __shfl_xor_sync(0xffffffffu, s, d);
        const int ow = __shfl_xor_sync(0xffffffffu, word, d);
        if (greedy) {
          word = om > m || (om == m && ow < word) ? ow : word;
          m = fmaxf(m, om);
        } else {
          const float m_new = fmaxf(m, om), ref = fmaxf(m_new, -3.4028235e38f);
          s = s * ex2((m - ref) * per_unit_log2) + os * ex2((om - ref) * per_unit_log2);
          m = m_new;
        }
      }
      if (lane == 0) s_part[count][warp] = make_uint2(__float_as_uint(m), greedy ? static_cast<uint32_t>(word) : __float_as_uint(s));
    }
    __syncthreads();
    auto join = [&](const uint2* parts, int many, float& m, uint32_t& second) {
      m = -CUDART_INF_F;
      for (int i = 0; i < many; ++i) m = fmaxf(m, __uint_as_float(parts[i].x));
      if (greedy) {
        second = 0x7fffffffu;
        for (int i = 0; i < many; ++i)
          if (__uint_as_float(parts[i].x) == m) second = min(second, parts[i].y);
      } else {
        const float ref = fmaxf(m, -3.4028235e38f);
        float s = 0.f;
        for (int i = 0; i < many; ++i) s += __uint_as_float(parts[i].y) * ex2((__uint_as_float(parts[i].x) - ref) * per_unit_log2);
        second = __float_as_uint(s);
      }
    };
    if (warp < count) {
      float m;
      uint32_t second;
      join(s_part[warp], kVerifyWarps, m, second);
      if (lane < p.cluster) put_peer(&s_all[turn][warp][rank], lane, make_uint2(__float_as_uint(m), second));
    }
    cluster_sync();
    // ---- the walk over the window ----
    for (int k = 0; k < count && walking; ++k) {
      uint32_t second;
      join(s_all[turn][k], p.cluster, top, second);
      const int node_was = node;
      int largest = -1;  // greedy: the token
      if (greedy) {
        best_word = static_cast<int>(second);
        if (top > -CUDART_INF_F) {
          const Row<T> row(logits + node * p.logits_stride, p.vocab);
          const uint4 raw = row.raw(best_word);
          const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
          for (int i = kN - 1; i >= 0; --i)
            if (number(x[i]) == top) largest = best_word * kN - row.skip + i;
        }
      }
      double sum = __uint_as_float(second);
      // a first look with the sum of 32 bits; where that could err, again with the sum of 64
      for (int look = 0; look < 2; ++look) {
        if (warp == 0) {
          const double u = greedy ? 0.0 : static_cast<double>(s_coin[node]);
          double mass = 0.0;
          int taken = 0, unsure = look == 0 && !greedy && !(sum >= 0.5 && sum < 1e30);
          for (int i0 = node + 1 - (node + 1) % 32; i0 < n && !taken && !unsure; i0 += 32) {
            const int i = i0 + lane;
            const bool child = i < n && i > node && s_parent[i] == node && s_token[i] >= 0;
            bool take, close;
            if (greedy) {
              take = child && s_token[i] == largest;
              close = false;
            } else {
              const double w = child && !s_again[i] && top > -CUDART_INF_F ? weight(s_x[i], top, per_unit) : 0.0;
              double left, right;
              if (probs) {
                left = u * static_cast<double>(child ? s_q[i] : 0.f) * sum;
                right = w;
              } else {
                double run = w;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                  const double below = __shfl_up_sync(0xffffffffu, run, d);
                  if (lane >= d) run += below;
                }
                left = u * sum;
                right = mass + run;
                mass += __shfl_sync(0xffffffffu, run, 31);
              }
              take = child && !s_again[i] && w > 0.0 && left < right;
              close = look == 0 && child && fabs(left - right) <= 1e-5 * (left + right);
            }
            const unsigned first = __ballot_sync(0xffffffffu, take), near_one = __ballot_sync(0xffffffffu, close);
            // (one that is near decides only if none ahead of it was taken)
            if (near_one && (!first || __ffs(near_one) <= __ffs(first))) unsure = 1;
            else if (first) taken = i0 + __ffs(first) - 1;
          }
          if (lane == 0) s_next = unsure ? -1 : taken;
        }
        __syncthreads();
        const int next = s_next;
        __syncthreads();
        if (next >= 0) {
          if (next > 0) {
            node = next;
            ++accepted;
            if (tid == 0) s_path[accepted] = next;
          }
          break;
        }
        sum = exact_sum(node, top);
      }
      if (node == node_was) walking = false;                        // the row that the sequence ends with
      else if (k + 1 >= count || node != s_first[node_was]) break;  // beyond the window
      if (greedy) s_last = largest;  // (the same in all threads)
    }
    turn ^= 1;
  }

  // ---- the token behind the last accepted row ----
  if (greedy) {
    // s_last is of the last row looked at
  } else if (top == -CUDART_INF_F) {
    if (tid == 0) s_last = -1;
  } else {
    const Row<T> row(logits + node * p.logits_stride, p.vocab);
    const bool rejected = s_first[node] < n;
    const float* q = rejected && probs ? probs + node * p.probs_stride : nullptr;
    const bool without = rejected && !probs;
    const double sum = q ? exact_sum(node, top) : 1.0;
    if (warp == 0) {
      int many = 0;
      for (int i0 = 0; without && i0 < n; i0 += 32) {
        const int i = i0 + lane;
        const bool kid = i < n && s_parent[i] == node && s_token[i] >= 0;
        const unsigned kids = __ballot_sync(0xffffffffu, kid);
        if (kid) s_kids[many + __popc(kids & ((1u << lane) - 1))] = s_token[i];
        many += __popc(kids);
      }
      if (lane == 0) s_num_kids = many;
    }
    __syncthreads();
    const int w0 = begin_of(row, my_warp), w1 = begin_of(row, my_warp + 1);
    bool kids_here = false;  // in the warp's run
    for (int j = 0; j < s_num_kids; ++j) kids_here |= s_kids[j] >= w0 * kN - row.skip && s_kids[j] < w1 * kN - row.skip;
    bool plain = false;  // nothing left of what was asked for: from p itself
    auto part = [&](int first, const T* x, double (&w)[kN]) {
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        w[k] = weight(number(x[k]), top, per_unit);
        const int i = first + k;
        if (!plain && q && w[k] > 0.0) w[k] = fmax(w[k] / sum - static_cast<double>(q[i]), 0.0);
      }
      if (!plain && kids_here) {
        for (int j = 0; j < s_num_kids; ++j) {
          const int at = s_kids[j] - first;
#pragma unroll
          for (int k = 0; k < kN; ++k)
            if (k == at) w[k] = 0.0;
        }
      }
    };
    double whole;
    for (int look = 0; look < 2; ++look) {
      double mine = 0.0;
      over(row, w0, w1, [&](int first, const T* x) {
        double w[kN];
        part(first, x, w);
#pragma unroll
        for (int k = 0; k < kN; ++k) mine += w[k];
      });
      whole = cluster_sum(mine);
      if (whole > 0.0 || plain) break;
      plain = true;
    }
    // the warp whose run of the vocabulary the threshold falls into, all threads alike
    const double threshold = static_cast<double>(p.draws[b]) * whole;
    double below = 0.0, behind = 0.0;
    int block = -1;
    turn_sum ^= 1;  // the sums that were exchanged last
    for (int r = 0; r < p.cluster; ++r) {
      const double s = s_sums[turn_sum][r];
      if (s > 0.0 && (block < 0 || below + behind <= threshold)) {
        block = r;
        below += behind;
        behind = s;
      }
    }
    if (block == rank) {
      int which = -1;
      double at = below;
      behind = 0.0;
      for (int w = 0; w < kVerifyWarps; ++w) {
        const double s = s_sum[w];
        if (s > 0.0 && (which < 0 || at + behind <= threshold)) {
          which = w;
          at += behind;
          behind = s;
        }
      }
      if (warp == which) {
        int found = -1, last = -1;  // the first past the threshold; the last with any weight
        for (int c0 = w0; c0 < w1 && found < 0; c0 += 32) {
          double w[kN], run = 0.0;
#pragma unroll
          for (int k = 0; k < kN; ++k) w[k] = 0.0;
          const int first = (c0 + lane) * kN - row.skip;
          if (c0 + lane < w1) {
            const uint4 raw = row.raw(c0 + lane);
            part(first, reinterpret_cast<const T*>(&raw), w);
          }
#pragma unroll
          for (int k = 0; k < kN; ++k) run += w[k];
          const double own = run;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const double o = __shfl_up_sync(0xffffffffu, run, d);
            if (lane >= d) run += o;
          }
          double here = at + run - own;
          int candidate = -1, any = -1;
#pragma unroll
          for (int k = 0; k < kN; ++k) {
            here += w[k];
            if (w[k] > 0.0) {
              any = first + k;
              if (candidate < 0 && here > threshold) candidate = first + k;
            }
          }
          const unsigned hit = __ballot_sync(0xffffffffu, candidate >= 0), some = __ballot_sync(0xffffffffu, any >= 0);
          if (hit) found = __shfl_sync(0xffffffffu, candidate, __ffs(hit) - 1);
          if (some) last = __shfl_sync(0xffffffffu, any, 31 - __clz(some));
          at += __shfl_sync(0xffffffffu, run, 31);
        }
        if (lane == 0) out_tokens[accepted] = found >= 0 ? found : last;
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

}  // namespace

int draft_tree(int* positions, long long* visible, const int* parents, const int* cu, const int* lengths, int batch, int num_tokens, int max_seqlen, void* stream) {
  if (batch == 0 || num_tokens == 0 || max_seqlen == 0) return QS_OK;
  const int threads = (max_seqlen + 31) / 32 * 32, words = (max_seqlen + 63) / 64;
  return paged::launch(tree_kernel, dim3(batch), threads, 0, stream, "draft_tree", 1, positions, reinterpret_cast<unsigned long long*>(visible), parents, cu, lengths, num_tokens,
                       max_seqlen, words);
}

int verify_drafts(const VerifyArgs& a) {
  if (a.batch == 0 || a.max_seqlen == 0) return QS_OK;
  VerifyParams p{};
  p.logits = a.logits; p.logits_stride = a.logits_stride; p.probs_stride = a.probs_stride; p.tokens = a.tokens; p.parents = a.parents; p.probs = a.probs; p.cu = a.cu_seqlens;
  p.coins = a.coins; p.draws = a.draws; p.temperatures = a.temperatures; p.out_tokens = a.out_tokens; p.out_rows = a.out_rows; p.out_counts = a.out_counts;
  p.num_tokens = a.num_tokens; p.vocab = a.vocab; p.max_seqlen = a.max_seqlen;
  p.cluster = kMostBlocks;
  p.log2_warps = 7;
  const dim3 grid(static_cast<unsigned>(a.batch) * p.cluster);
  auto run = [&](auto kern) { return paged::launch(kern, grid, kVerifyThreads, 0, a.stream, "verify_drafts", p.cluster, p); };
  return a.type == 0 ? run(verify_kernel<__half>) : a.type == 1 ? run(verify_kernel<__nv_bfloat16>) : run(verify_kernel<float>);
}

}  // namespace qs
