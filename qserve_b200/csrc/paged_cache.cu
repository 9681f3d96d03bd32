// qserve_b200 -- portions of sequences into and out of the paged INT4 / INT8 key/value cache.
//
// append: token i of sequence b's portion of n_b takes position p = lengths[b] - n_b + i.  Queries and keys are rotated (entry i with entry i + 64, angle
// p base^(-2 i / 128)), keys and values quantised per (token, kv head): scale s = half((max - min) / L), zero z = half(-L min / (max - min)), code
// clamp(round(x / s + z), 0, L), L = 15 or 255.
// read: the same positions out of the pages again, as fp16; zeros for a row that has none.
#include <math_constants.h>

#include <cmath>
#include <type_traits>

#include "paged_common.cuh"

namespace qs {
namespace {

using namespace paged;

constexpr int kWarps = 4;

// Turns per position of the 64 pairs.  The angle of a far position has lost all its low bits as an fp32 product (position 100000, pair 1: 0.01 rad), so the turns are
// taken in 64 bits, their whole part dropped, and sine and cosine rounded to fp32 once.
struct Turns {
  double per_position[kD / 2];
};

// Eight lanes hold a row: lane l of them elements 8 l .. and 64 + 8 l .. as fp32 pairs.
constexpr uint32_t kMagic = 0x4b400000u;  // the bits of 1.5 x 2^23: a sum with it has a small whole number in its low bits, rounded to even
__device__ __forceinline__ f2 both(float x) { return pack2(x, x); }
// two products, each rounded: one by one, because the compiler makes a fused operation of a packed product and the sum after it, rounding modifiers or not (7 of 10^6
// INT8 codes were others than the definition's)
__device__ __forceinline__ f2 product(f2 a, f2 b) {
  const float2 x = unpack2(a), y = unpack2(b);
  return pack2(__fmul_rn(x.x, y.x), __fmul_rn(x.y, y.y));
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
  float y;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// the row's scale and zero and this lane's codes: INT4 word w of dims 64 w + 8 l .., INT8 words 2 w and 2 w + 1
template <int BITS>
struct Quantised {
  __half scale, zero;
  uint32_t word[BITS / 2];
};
template <int BITS>
__device__ __forceinline__ Quantised<BITS> quantise_row(const f2 (&x)[8]) {
  constexpr float kTop = BITS == 4 ? 15.f : 255.f;
  float hi, lo;
  {
    const float2 a = unpack2(x[0]);
    hi = max3_nan(a.x, a.y, a.y);
    lo = min3_nan(a.x, a.y, a.y);
#pragma unroll
    for (int j = 1; j < 8; ++j) {
      const float2 b = unpack2(x[j]);
      hi = max3_nan(hi, b.x, b.y);
      lo = min3_nan(lo, b.x, b.y);
    }
  }
#pragma unroll
  for (int m = 4; m >= 1; m >>= 1) {
    const float h = __shfl_xor_sync(0xffffffffu, hi, m), w = __shfl_xor_sync(0xffffffffu, lo, m);
    hi = max3_nan(hi, h, h);
    lo = min3_nan(lo, w, w);
  }
  Quantised<BITS> r;
  const float span = __fsub_rn(hi, lo);
  r.scale = __float2half_rn(__fdiv_rn(span, kTop));
  r.zero = __float2half_rn(__fdiv_rn(__fmul_rn(-kTop, lo), span));
  float s = __half2float(r.scale), z = __half2float(r.zero), inv = __fdiv_rn(1.f, s);
  if (!(span <= 131008.f)) {  // a number that is none, or has no end: the whole row reads as NaN
    r.scale = r.zero = __ushort_as_half(0x7fffu);
    inv = z = 0.f;
  } else if (s == 0.f || !(fabsf(z) <= 65504.f)) {
    // values of one kind, or so near to one another that their zero is none in fp16: the middle c of the row, held as 1 x |c| or as 0 - 1 x |c|
    const float c = __half2float(__float2half_rn((hi + lo) * 0.5f));
    r.scale = __float2half_rn(fabsf(c));
    r.zero = __float2half_rn(c < 0.f ? 1.f : 0.f);
    inv = 0.f;
    z = c > 0.f ? 1.f : 0.f;
  } else if (fmaxf(hi, -lo) > 65000.f) {
    // A row that reaches the ends of fp16, whose rounded scale and zero may take its first or its last code past them: the scale is rounded down then, and if that is not enough the
    // zero goes to the next number towards the other end.  (All pairs of least and largest number with one above 65000 tried on the CPU: 145000 of 4 million are past the ends as
    // rounded, 798 with the scale rounded down, none with the zero moved; and none of those that stay below.)
    bool below, above;
    auto ends = [&] {
      if constexpr (BITS == 4) {
        const __half c = __float2half_rn(-__fmul_rn(s, z));
        below = __half_as_ushort(c) == 0xfc00u;
        above = fmaf(s, kTop, __half2float(c)) >= 65520.f;  // (65520 is the least number that rounds to infinity)
      } else {
        below = __fmul_rn(s, z) >= 65520.f;
        above = __fmul_rn(s, kTop - z) >= 65520.f;
      }
    };
    ends();
    if (below || above) {
      r.scale = __float2half_rd(__fdiv_rn(span, kTop));
      s = __half2float(r.scale);
      ends();
      if (below || above) {
        const int bits = __half_as_ushort(r.zero), next = ((bits & 0x8000) ? -(bits & 0x7fff) : bits) + (below ? -1 : 1);
        r.zero = __ushort_as_half(static_cast<unsigned short>(next < 0 ? 0x8000 - next : next));
        z = __half2float(r.zero);
      }
      inv = __fdiv_rn(1.f, s);
    }
  }
#pragma unroll
  for (int k = 0; k < BITS / 2; ++k) r.word[k] = 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // x / s + z with both roundings, kept to 0 .. top, then to the nearest whole number
    const float2 t = unpack2(add2(product(x[j], both(inv)), both(z)));
    const float2 c = unpack2(add2(pack2(fminf(fmaxf(t.x, 0.f), kTop), fminf(fmaxf(t.y, 0.f), kTop)), both(__uint_as_float(kMagic))));
    constexpr int kPer = 32 / BITS;  // codes of a word
    uint32_t& w = r.word[2 * j / kPer];
    w += (__float_as_uint(c.x) << (BITS * (2 * j % kPer))) + (__float_as_uint(c.y) << (BITS * (2 * j % kPer + 1)));
  }
  // the constant's bits, once for all codes of a word
  constexpr uint32_t kBias = BITS == 4 ? kMagic * 0x11111111u : kMagic * 0x01010101u;
#pragma unroll
  for (int k = 0; k < BITS / 2; ++k) r.word[k] -= kBias;
  return r;
}

struct AppendParams {
  const __half *q, *k, *v;
  __half* q_out;
  long long q_stride, k_stride, v_stride, q_out_stride;
  const long long* kv_pointers;
  const int *cu, *lengths;
  int batch, num_tokens, max_blocks, num_heads, num_kv_heads, rows_per_warp;
  Turns turns;
};

// A warp per token and run of its head rows, four rows at a time with eight lanes each.  ROWS: groups of four rows whose loads are on their way together.
template <int BITS, int ROWS>
__global__ void __launch_bounds__(32 * kWarps) append_kernel(const __grid_constant__ AppendParams p) {
  using G = Geom<BITS>;
  __shared__ __align__(16) float s_cos[kWarps][kD / 2], s_sin[kWarps][kD / 2];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, l = lane & 7;
  const int t = blockIdx.x * kWarps + warp;
  if (t >= p.num_tokens) return;
  const int rows = p.num_heads + 2 * p.num_kv_heads, rotated = p.num_heads + p.num_kv_heads;
  const int begin = blockIdx.y * p.rows_per_warp, end = min(rows, begin + p.rows_per_warp);
  auto source = [&](int r) {
    if (r < p.num_heads) return p.q + t * p.q_stride + r * kD;
    if (r < rotated) return p.k + t * p.k_stride + (r - p.num_heads) * kD;
    return p.v + t * p.v_stride + (r - rotated) * kD;
  };
  uint4 lo[ROWS], hi[ROWS];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int e = 0; e < ROWS; ++e) {
      const int r = r0 + 4 * e + sub;
      lo[e] = hi[e] = make_uint4(0u, 0u, 0u, 0u);
      if (r < end) {
        const uint4* x = reinterpret_cast<const uint4*>(source(r)) + l;
        lo[e] = x[0];
        hi[e] = x[8];
      }
    }
  };
  fetch(begin);  // ahead of the tables: they come one after the other
  const int b = sequence_of(p.cu, p.batch, t);
  if (b < 0) return;
  const Portion portion = portion_of(p.cu, p.lengths, b, p.num_tokens);
  const int pos = portion.first + t - portion.start;
  const int block = pos >> 6, slot = pos & (kPage - 1);
  const bool held = pos >= 0 && block < p.max_blocks;  // a position outside the sequence's pages goes nowhere
  uint8_t* pages[2] = {nullptr, nullptr};
  if (held && end > p.num_heads) {
    const long long* table = p.kv_pointers + static_cast<long long>(b) * 2 * p.max_blocks + block;
    pages[0] = reinterpret_cast<uint8_t*>(table[0]);
    pages[1] = reinterpret_cast<uint8_t*>(table[p.max_blocks]);
  }
  if (begin < rotated) {
#pragma unroll
    for (int i = lane; i < kD / 2; i += 32) {
      const double turns = p.turns.per_position[i] * pos;
      double sn, cs;
      sincospi(2.0 * (turns - rint(turns)), &sn, &cs);
      s_sin[warp][i] = static_cast<float>(sn);
      s_cos[warp][i] = static_cast<float>(cs);
    }
    __syncwarp();
  }
  for (int r0 = begin; r0 < end; r0 += 4 * ROWS) {
    if (r0 > begin) fetch(r0);
#pragma unroll
    for (int e = 0; e < ROWS; ++e) {
      if (r0 + 4 * e >= end) break;
      const int r = r0 + 4 * e + sub;
      const bool live = r < end;
      f2 x[8];
      {
        const __half2* a = reinterpret_cast<const __half2*>(&lo[e]);
        const __half2* c = reinterpret_cast<const __half2*>(&hi[e]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __half22float2(a[j]), g = __half22float2(c[j]);
          x[j] = pack2(f.x, f.y);
          x[4 + j] = pack2(g.x, g.y);
        }
      }
      if (live && r < rotated) {
        uint4 out[2];
        __half2* o = reinterpret_cast<__half2*>(out);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const ulonglong2 cs = *reinterpret_cast<const ulonglong2*>(&s_cos[warp][8 * l + 2 * j]), sn = *reinterpret_cast<const ulonglong2*>(&s_sin[warp][8 * l + 2 * j]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const f2 c = k ? cs.y : cs.x, s = k ? sn.y : sn.x, f0 = x[j + k], f1 = x[4 + j + k];
            x[j + k] = fma2(product(s, f1), both(-1.f), product(c, f0));
            x[4 + j + k] = add2(product(c, f1), product(s, f0));
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 f = unpack2(x[j]);
          o[j] = __floats2half2_rn(f.x, f.y);
        }
        if (r < p.num_heads) {
          uint4* dst = reinterpret_cast<uint4*>(p.q_out + t * p.q_out_stride + r * kD) + l;
          dst[0] = out[0];
          dst[8] = out[1];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {  // keys are quantised as fp16 numbers
            const float2 f = __half22float2(o[j]);
            x[j] = pack2(f.x, f.y);
          }
        }
      }
      const bool mine = live && held && r >= p.num_heads;
      if (!__any_sync(0xffffffffu, mine)) continue;
      const Quantised<BITS> c = quantise_row<BITS>(x);
      if (!mine) continue;
      const int which = r >= rotated, head = r - p.num_heads - which * p.num_kv_heads;
      uint8_t* page = which ? pages[1] : pages[0];
      uint8_t* row = page + G::codes_at(head) + slot * G::kRow;
      if constexpr (BITS == 4) {
        reinterpret_cast<uint32_t*>(row)[l] = c.word[0];
        reinterpret_cast<uint32_t*>(row)[8 + l] = c.word[1];
      } else {
        reinterpret_cast<uint2*>(row)[l] = make_uint2(c.word[0], c.word[1]);
        reinterpret_cast<uint2*>(row)[8 + l] = make_uint2(c.word[2], c.word[3]);
      }
      if (l == 0) {
        *reinterpret_cast<__half*>(page + G::scales_at(head, p.num_kv_heads) + slot * 2) = c.scale;
        *reinterpret_cast<__half*>(page + G::zeros_at(head, p.num_kv_heads) + slot * 2) = c.zero;
      }
    }
  }
}

struct ReadParams {
  __half *k, *v;
  const long long* kv_pointers;
  const int *cu, *lengths;
  int batch, num_tokens, max_blocks, num_kv_heads;
};

// A warp per token and run of 4 ROWS head rows, eight lanes a row: lane l has dims 8 l .. and 64 + 8 l .., so that a store takes whole sectors; everything that the
// warp reads of the pages is on its way together.
template <int BITS, int ROWS>
__global__ void __launch_bounds__(32 * kWarps) read_kernel(const ReadParams p) {
  using G = Geom<BITS>;
  using Word = std::conditional_t<BITS == 4, uint32_t, uint2>;  // eight codes
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane >> 3, l = lane & 7;
  const int t = blockIdx.x * kWarps + warp;
  if (t >= p.num_tokens) return;
  const int b = sequence_of(p.cu, p.batch, t);
  if (b < 0) return;
  const Portion portion = portion_of(p.cu, p.lengths, b, p.num_tokens);
  const int pos = portion.first + t - portion.start;
  const int block = pos >> 6, slot = pos & (kPage - 1);
  const bool held = pos >= 0 && block < p.max_blocks;  // a row without a position gets zeros, as attention gives it
  const uint8_t* pages[2] = {nullptr, nullptr};
  if (held) {
    const long long* table = p.kv_pointers + static_cast<long long>(b) * 2 * p.max_blocks + block;
    pages[0] = reinterpret_cast<const uint8_t*>(table[0]);
    pages[1] = reinterpret_cast<const uint8_t*>(table[p.max_blocks]);
  }
  Word lo[ROWS], hi[ROWS];
  __half s[ROWS], z[ROWS];
  const int r0 = blockIdx.y * 4 * ROWS + sub;
#pragma unroll
  for (int e = 0; e < ROWS; ++e) {
    const int r = r0 + 4 * e, which = r >= p.num_kv_heads, head = r - which * p.num_kv_heads;
    lo[e] = hi[e] = Word{};
    s[e] = z[e] = __ushort_as_half(0);
    if (r < 2 * p.num_kv_heads && held) {
      const uint8_t* page = which ? pages[1] : pages[0];
      const Word* row = reinterpret_cast<const Word*>(page + G::codes_at(head) + slot * G::kRow);
      lo[e] = row[l];
      hi[e] = row[8 + l];
      s[e] = *reinterpret_cast<const __half*>(page + G::scales_at(head, p.num_kv_heads) + slot * 2);
      z[e] = *reinterpret_cast<const __half*>(page + G::zeros_at(head, p.num_kv_heads) + slot * 2);
    }
  }
#pragma unroll
  for (int e = 0; e < ROWS; ++e) {
    const int r = r0 + 4 * e, which = r >= p.num_kv_heads, head = r - which * p.num_kv_heads;
    if (r >= 2 * p.num_kv_heads) break;
    uint4* dst = reinterpret_cast<uint4*>((which ? p.v : p.k) + (static_cast<long long>(t) * p.num_kv_heads + head) * kD);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const Word w = half ? hi[e] : lo[e];
      uint4 out;
      __half2* o = reinterpret_cast<__half2*>(&out);
      if constexpr (BITS == 4) {
        const __half2 s2 = __half2half2(s[e]), c2 = __half2half2(__hmul(__hneg(s[e]), z[e]));
        __half2 u[4], x[4];
        codes_of_word4(w, u);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __hfma2(u[j], s2, c2);
        o[0] = __lows2half2(x[0], x[1]);
        o[1] = __lows2half2(x[2], x[3]);
        o[2] = __highs2half2(x[0], x[1]);
        o[3] = __highs2half2(x[2], x[3]);
      } else {
        const float sf = __half2float(s[e]), zf = __half2float(z[e]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x = (i < 2 ? w.x : w.y) >> (16 * (i & 1));
          o[i] = __floats2half2_rn(sf * (static_cast<float>(x & 255u) - zf), sf * (static_cast<float>((x >> 8) & 255u) - zf));
        }
      }
      dst[8 * half + l] = out;
    }
  }
}

}  // namespace

int append_kv_cache(const AppendArgs& a) {
  if (a.num_tokens == 0 || a.batch == 0) return QS_OK;
  AppendParams p{};
  p.q = static_cast<const __half*>(a.q); p.k = static_cast<const __half*>(a.k); p.v = static_cast<const __half*>(a.v); p.q_out = static_cast<__half*>(a.q_out);
  p.q_stride = a.q_stride; p.k_stride = a.k_stride; p.v_stride = a.v_stride; p.q_out_stride = a.q_out_stride;
  p.kv_pointers = a.cache.kv_pointers; p.cu = a.cache.cu_seqlens; p.lengths = a.cache.lengths;
  p.batch = a.batch; p.num_tokens = a.num_tokens; p.max_blocks = a.cache.max_blocks; p.num_heads = a.num_heads; p.num_kv_heads = a.cache.num_kv_heads;
  const double step = std::pow(static_cast<double>(a.rotary_base), -2.0 / kD);
  double f = 0.15915494309189533577;  // 1 / (2 pi)
  for (int i = 0; i < kD / 2; ++i, f *= step) p.turns.per_position[i] = f;
  const int rows = p.num_heads + 2 * p.num_kv_heads, blocks = (a.num_tokens + kWarps - 1) / kWarps;
  // A token's rows are shared out over several warps, eight rows each at least, as long as that makes no more than 48 warps per multiprocessor: every one of them
  // works out the position's sines
  const long long fair = static_cast<long long>(rows) * a.num_tokens / (48 * num_sms());
  p.rows_per_warp = static_cast<int>(fair >= rows ? rows : 8 * (fair / 8 + 1));
  const dim3 grid(blocks, (rows + p.rows_per_warp - 1) / p.rows_per_warp);
  auto run = [&](auto kern) { return launch(kern, grid, 32 * kWarps, 0, a.stream, "append_kv_cache", 1, p); };
  return a.cache.int4 ? run(append_kernel<4, 2>) : run(append_kernel<8, 2>);
}

int read_kv_cache(void* k_out, void* v_out, const PagedCache& c, int batch, int num_tokens, void* stream) {
  if (num_tokens == 0 || batch == 0) return QS_OK;
  ReadParams p{};
  p.k = static_cast<__half*>(k_out); p.v = static_cast<__half*>(v_out); p.kv_pointers = c.kv_pointers; p.cu = c.cu_seqlens; p.lengths = c.lengths;
  p.batch = batch; p.num_tokens = num_tokens; p.max_blocks = c.max_blocks; p.num_kv_heads = c.num_kv_heads;
  constexpr int kRows = 4;
  const dim3 grid((num_tokens + kWarps - 1) / kWarps, (2 * c.num_kv_heads + 4 * kRows - 1) / (4 * kRows));
  auto run = [&](auto kern) { return launch(kern, grid, 32 * kWarps, 0, stream, "read_kv_cache", 1, p); };
  return c.int4 ? run(read_kernel<4, kRows>) : run(read_kernel<8, kRows>);
}

}  // namespace qs
