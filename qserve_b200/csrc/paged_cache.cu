// qserve_b200 -- portions of sequences into and out of the paged INT4 / INT8 key/value cache.
//
// append: token i of sequence b's portion of n_b takes position p = lengths[b] - n_b + i.  Queries and keys are rotated (entry i with entry i + 64, angle
// p base^(-2 i / 128)), keys and values quantised per (token, kv head): scale s = half((max - min) / L), zero z = half(-L min / (max - min)), code
// clamp(round(x / s + z), 0, L), L = 15 or 255.
// read: the same positions out of the pages again, as fp16.
#include <math_constants.h>

#include <cmath>

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

// Eight lanes hold a row: lane l of them elements 8 l .. and 64 + 8 l .. as fp32 numbers.
struct Quantised {
  __half scale, zero;
  uint32_t code[16];
};
template <int BITS>
__device__ __forceinline__ Quantised quantise_row(const float (&x)[16]) {
  constexpr float kTop = BITS == 4 ? 15.f : 255.f;
  float hi = x[0], lo = x[0], poison = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    hi = fmaxf(hi, x[j]);
    lo = fminf(lo, x[j]);
    poison = fmaf(x[j], 0.f, poison);  // NaN where the row has a number that is none or has no end
  }
#pragma unroll
  for (int m = 4; m >= 1; m >>= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    poison += __shfl_xor_sync(0xffffffffu, poison, m);
  }
  Quantised r;
  const float span = __fsub_rn(hi, lo);
  r.scale = __float2half_rn(__fdiv_rn(span, kTop));
  r.zero = __float2half_rn(__fdiv_rn(__fmul_rn(-kTop, lo), span));
  const float s = __half2float(r.scale);
  float z = __half2float(r.zero);
  if (poison != 0.f) {  // NaN: the whole row reads as NaN
    r.scale = r.zero = __ushort_as_half(0x7fffu);
#pragma unroll
    for (int j = 0; j < 16; ++j) r.code[j] = 0u;
  } else if (s == 0.f || !(fabsf(z) <= 65504.f)) {
    // values of one kind, or so near to one another that their zero is none in fp16: the middle c of the row, held as 1 x |c| or as 0 - 1 x |c|
    const float c = __half2float(__float2half_rn((hi + lo) * 0.5f));
    r.scale = __float2half_rn(fabsf(c));
    r.zero = __float2half_rn(c < 0.f ? 1.f : 0.f);
#pragma unroll
    for (int j = 0; j < 16; ++j) r.code[j] = c > 0.f ? 1u : 0u;
  } else {
    const float inv = __fdiv_rn(1.f, s);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      asm("cvt.rni.sat.u8.f32 %0, %1;" : "=r"(r.code[j]) : "f"(__fadd_rn(__fmul_rn(x[j], inv), z)));
      if constexpr (BITS == 4) r.code[j] = min(r.code[j], 15u);
    }
  }
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
  const int b = sequence_of(p.cu, p.batch, t);
  if (b < 0) return;
  const Portion portion = portion_of(p.cu, p.lengths, b, p.num_tokens);
  const int pos = portion.first + t - portion.start;
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
      if (r < end) {
        const uint4* x = reinterpret_cast<const uint4*>(source(r)) + l;
        lo[e] = x[0];
        hi[e] = x[8];
      }
    }
  };
  fetch(begin);
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
  const int block = pos >> 6, slot = pos & (kPage - 1);
  const bool held = pos >= 0 && block < p.max_blocks;  // a position outside the sequence's pages goes nowhere
  for (int r0 = begin; r0 < end; r0 += 4 * ROWS) {
    if (r0 > begin) fetch(r0);
#pragma unroll
    for (int e = 0; e < ROWS; ++e) {
      if (r0 + 4 * e >= end) break;
      const int r = r0 + 4 * e + sub;
      const bool live = r < end;
      float x[16];
      {
        const __half2* a = reinterpret_cast<const __half2*>(&lo[e]);
        const __half2* c = reinterpret_cast<const __half2*>(&hi[e]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = __half22float2(a[j]), g = __half22float2(c[j]);
          x[2 * j] = live ? f.x : 0.f; x[2 * j + 1] = live ? f.y : 0.f;
          x[8 + 2 * j] = live ? g.x : 0.f; x[8 + 2 * j + 1] = live ? g.y : 0.f;
        }
      }
      if (live && r < rotated) {
        float cs[8], sn[8];
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const float4 c = *reinterpret_cast<const float4*>(&s_cos[warp][8 * l + j]), s = *reinterpret_cast<const float4*>(&s_sin[warp][8 * l + j]);
          cs[j] = c.x; cs[j + 1] = c.y; cs[j + 2] = c.z; cs[j + 3] = c.w;
          sn[j] = s.x; sn[j + 1] = s.y; sn[j + 2] = s.z; sn[j + 3] = s.w;
        }
        uint4 out[2];
        __half2* o = reinterpret_cast<__half2*>(out);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float f0 = x[j], f1 = x[8 + j];
          x[j] = __fsub_rn(__fmul_rn(cs[j], f0), __fmul_rn(sn[j], f1));
          x[8 + j] = __fadd_rn(__fmul_rn(cs[j], f1), __fmul_rn(sn[j], f0));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          o[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
          const float2 f = __half22float2(o[j]);  // keys are quantised as fp16 numbers
          x[2 * j] = f.x;
          x[2 * j + 1] = f.y;
        }
        if (r < p.num_heads) {
          uint4* dst = reinterpret_cast<uint4*>(p.q_out + t * p.q_out_stride + r * kD) + l;
          dst[0] = out[0];
          dst[8] = out[1];
        }
      }
      const bool mine = live && held && r >= p.num_heads;
      if (!__any_sync(0xffffffffu, mine)) continue;
      const Quantised c = quantise_row<BITS>(x);
      if (!mine) continue;
      const int which = r >= rotated, head = r - p.num_heads - which * p.num_kv_heads;
      uint8_t* page = reinterpret_cast<uint8_t*>(p.kv_pointers[(static_cast<long long>(b) * 2 + which) * p.max_blocks + block]);
      uint8_t* row = page + G::codes_at(head) + slot * G::kRow;
      if constexpr (BITS == 4) {
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j >> 3] |= c.code[j] << (4 * (j & 7));
        reinterpret_cast<uint32_t*>(row)[l] = w[0];
        reinterpret_cast<uint32_t*>(row)[8 + l] = w[1];
      } else {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j >> 2] |= c.code[j] << (8 * (j & 3));
        reinterpret_cast<uint2*>(row)[l] = make_uint2(w[0], w[1]);
        reinterpret_cast<uint2*>(row)[8 + l] = make_uint2(w[2], w[3]);
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

// A warp per token, eight lanes per head row: 16 codes and 32 bytes of results a lane.
template <int BITS>
__global__ void __launch_bounds__(32 * kWarps) read_kernel(const ReadParams p) {
  using G = Geom<BITS>;
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
  if (pos < 0 || block >= p.max_blocks) return;
  const uint8_t* pages[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) pages[w] = reinterpret_cast<const uint8_t*>(p.kv_pointers[(static_cast<long long>(b) * 2 + w) * p.max_blocks + block]);
#pragma unroll 4
  for (int r = sub; r < 2 * p.num_kv_heads; r += 4) {
    const int which = r >= p.num_kv_heads, head = r - which * p.num_kv_heads;
    const uint8_t* page = which ? pages[1] : pages[0];
    const uint8_t* row = page + G::codes_at(head) + slot * G::kRow;
    const __half s = *reinterpret_cast<const __half*>(page + G::scales_at(head, p.num_kv_heads) + slot * 2);
    const __half z = *reinterpret_cast<const __half*>(page + G::zeros_at(head, p.num_kv_heads) + slot * 2);
    uint4 out[2];
    __half2* o = reinterpret_cast<__half2*>(out);
    if constexpr (BITS == 4) {
      const uint2 w = reinterpret_cast<const uint2*>(row)[l];
      const __half2 s2 = __half2half2(s), c2 = __half2half2(__hmul(__hneg(s), z));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        __half2 u[4], x[4];
        codes_of_word4(i ? w.y : w.x, u);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __hfma2(u[j], s2, c2);
        o[4 * i] = __lows2half2(x[0], x[1]);
        o[4 * i + 1] = __lows2half2(x[2], x[3]);
        o[4 * i + 2] = __highs2half2(x[0], x[1]);
        o[4 * i + 3] = __highs2half2(x[2], x[3]);
      }
    } else {
      const uint4 w = reinterpret_cast<const uint4*>(row)[l];
      const uint32_t words[4] = {w.x, w.y, w.z, w.w};
      const float sf = __half2float(s), zf = __half2float(z);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t x = words[i >> 1] >> (16 * (i & 1));
        o[i] = __floats2half2_rn(sf * (static_cast<float>(x & 255u) - zf), sf * (static_cast<float>((x >> 8) & 255u) - zf));
      }
    }
    __half* dst = (which ? p.v : p.k) + (static_cast<long long>(t) * p.num_kv_heads + head) * kD + 16 * l;
    reinterpret_cast<uint4*>(dst)[0] = out[0];
    reinterpret_cast<uint4*>(dst)[1] = out[1];
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
  const bool few = blocks < 2 * num_sms();  // a token's rows are shared out over several warps
  p.rows_per_warp = few ? 8 : rows;
  const dim3 grid(blocks, (rows + p.rows_per_warp - 1) / p.rows_per_warp);
  auto run = [&](auto kern) { return launch(kern, grid, 32 * kWarps, 0, a.stream, "append_kv_cache", 1, p); };
  if (a.cache.int4) return few ? run(append_kernel<4, 2>) : run(append_kernel<4, 4>);
  return few ? run(append_kernel<8, 2>) : run(append_kernel<8, 4>);
}

int read_kv_cache(void* k_out, void* v_out, const PagedCache& c, int batch, int num_tokens, void* stream) {
  if (num_tokens == 0 || batch == 0) return QS_OK;
  ReadParams p{};
  p.k = static_cast<__half*>(k_out); p.v = static_cast<__half*>(v_out); p.kv_pointers = c.kv_pointers; p.cu = c.cu_seqlens; p.lengths = c.lengths;
  p.batch = batch; p.num_tokens = num_tokens; p.max_blocks = c.max_blocks; p.num_kv_heads = c.num_kv_heads;
  const dim3 grid((num_tokens + kWarps - 1) / kWarps);
  auto run = [&](auto kern) { return launch(kern, grid, 32 * kWarps, 0, stream, "read_kv_cache", 1, p); };
  return c.int4 ? run(read_kernel<4>) : run(read_kernel<8>);
}

}  // namespace qs
