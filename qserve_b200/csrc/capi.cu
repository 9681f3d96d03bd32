// qserve_b200 -- extern "C" entry points (include/qserve_b200.h) and error plumbing.
#include <cstdarg>
#include <cstdio>

#include "../../include/qserve_b200.h"
#include "common.cuh"
#include "launch.h"

namespace qs {

static thread_local char g_err[1024] = "";
static int g_pdl = 1;
static int g_force_split = 0;
static int g_force_nt = 0;
static void* g_gemm_prof = nullptr;

int set_error(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int check_cuda(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return QS_OK;
  cudaGetLastError();  // clear the sticky launch error
  return set_error(QS_ERR_CUDA, "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
}

bool pdl_enabled() { return g_pdl != 0; }

int device_ordinal() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) dev = 0;
  return dev;
}
int num_sms() { return num_sms(device_ordinal()); }
int num_sms(int dev) {
  static int sms[kMaxDevices] = {};
  if (!sms[dev]) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    sms[dev] = n > 0 ? n : 148;
  }
  return sms[dev];
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace qs

using namespace qs;

extern "C" {

int qs_abi_version(void) { return QS_ABI_VERSION; }
const char* qs_last_error(void) { return g_err; }
int qs_set_pdl(int enabled) {
  const int old = g_pdl;
  g_pdl = enabled ? 1 : 0;
  return old;
}
int qs_gemm_force_tile_tokens(int nt) {
  const int old = g_force_nt;
  g_force_nt = nt;
  return old;
}

int qs_gemm_force_split(int split) {
  const int old = g_force_split;
  g_force_split = split;
  return old;
}
size_t qs_gemm_workspace_bytes(void) { return gemm_workspace_bytes(); }
int qs_set_trace_buffer(void* dev_buffer, unsigned capacity_records) {
  if (gemm_trace_install(dev_buffer, capacity_records) || attention_trace_install(dev_buffer, capacity_records) ||
      elementwise_trace_install(dev_buffer, capacity_records))
    return set_error(qs::QS_ERR_CUDA, "qs_set_trace_buffer: cudaMemcpyToSymbol failed");
  return 0;
}
int qs_gemm_set_profile_buffer(void* dev_buffer) {
  g_gemm_prof = dev_buffer;
  return 0;
}

int qs_w4a8_gemm_per_chn(const int8_t* in_feats, const int8_t* kernel, const void* wscales, const void* ascales, const void* w_szs,
                         const void* a_ssums, void* out_feats, int32_t* acc_out, int M, int N, int K, void* workspace, size_t workspace_bytes,
                         void* stream) {
  QS_REQUIRE(in_feats && kernel && wscales && ascales && w_szs && a_ssums && out_feats, "qgemm_w4a8_per_chn: null tensor");
  GemmArgs a;
  a.act = in_feats; a.weight = kernel; a.wscales = wscales; a.ascales = ascales; a.w_szs = w_szs; a.a_ssums = a_ssums;
  a.out = out_feats; a.acc_out = acc_out; a.M = M; a.N = N; a.K = K;
  a.workspace = workspace; a.workspace_bytes = workspace_bytes; a.force_split = g_force_split; a.force_nt = g_force_nt; a.prof = g_gemm_prof; a.stream = stream;
  return gemm_w4a8_per_chn(a);
}

int qs_w4a8_gemm_per_group(const int8_t* in_feats, const int8_t* kernel, const int8_t* zeros, const int8_t* scales_i8, const void* wscales,
                           const void* ascales, void* out_feats, int32_t* acc_out, int M, int N, int K, void* workspace,
                           size_t workspace_bytes, void* stream) {
  QS_REQUIRE(in_feats && kernel && zeros && scales_i8 && wscales && ascales && out_feats, "qgemm_w4a8_per_group: null tensor");
  QS_REQUIRE(aligned16(zeros) && aligned16(scales_i8), "qgemm_w4a8_per_group: level-2 scale/zero tensors must be 16-byte aligned");
  GemmArgs a;
  a.act = in_feats; a.weight = kernel; a.s2_zeros = zeros; a.s2_scales = scales_i8; a.wscales = wscales; a.ascales = ascales;
  a.out = out_feats; a.acc_out = acc_out; a.M = M; a.N = N; a.K = K;
  a.workspace = workspace; a.workspace_bytes = workspace_bytes; a.force_split = g_force_split; a.force_nt = g_force_nt; a.prof = g_gemm_prof; a.stream = stream;
  return gemm_w4a8_per_group(a);
}

int qs_w8a8_gemm(const int8_t* in_feats, const int8_t* kernel, const void* wscales, const void* ascales, void* out_feats, int32_t* acc_out,
                 int M, int N, int K, void* workspace, size_t workspace_bytes, void* stream) {
  QS_REQUIRE(in_feats && kernel && wscales && ascales && out_feats, "qgemm_w8a8: null tensor");
  GemmArgs a;
  a.act = in_feats; a.weight = kernel; a.wscales = wscales; a.ascales = ascales;
  a.out = out_feats; a.acc_out = acc_out; a.M = M; a.N = N; a.K = K;
  a.workspace = workspace; a.workspace_bytes = workspace_bytes; a.force_split = g_force_split; a.force_nt = g_force_nt; a.prof = g_gemm_prof; a.stream = stream;
  return gemm_w8a8(a);
}

size_t qs_attention_workspace_bytes(int batch, int num_heads, int head_dim) { return attention_workspace_bytes(batch, num_heads, head_dim, 32); }

int qs_single_query_attention(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                              const int64_t* kv_pointers, const int32_t* length_per_sample, void* out, int batch, int num_heads,
                              int num_kv_heads, int head_dim, int max_blocks_per_seq, int memory_max_seqlen, int tokens_per_block,
                              int size_per_token, int timestep, int rotary_embedding_dim, float rotary_base, int neox_rotary_style,
                              int int4_kv_cache, int kv_cache_with_zeros, void* workspace, size_t workspace_bytes, void* stream) {
  (void)neox_rotary_style;  // accepted and ignored: NeoX is hard-wired in the reference as well (fused_attention.cpp:109)
  QS_REQUIRE(q && k && v && kv_pointers && out, "single_query_attention: null tensor");
  DecodeAttnArgs a;
  a.q = q; a.k = k; a.v = v; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.kv_pointers = reinterpret_cast<const long long*>(kv_pointers); a.lengths = length_per_sample; a.out = out;
  a.batch = batch; a.num_heads = num_heads; a.num_kv_heads = num_kv_heads; a.head_dim = head_dim; a.max_blocks = max_blocks_per_seq;
  a.tokens_per_block = tokens_per_block; a.size_per_token = size_per_token; a.timestep = timestep; a.memory_max_len = memory_max_seqlen;
  a.rotary_dim = rotary_embedding_dim; a.rotary_base = rotary_base; a.int4_kv = int4_kv_cache; a.kv_zeros = kv_cache_with_zeros;
  a.workspace = workspace; a.workspace_bytes = workspace_bytes; a.prof = g_gemm_prof; a.stream = stream;
  return decode_attention(a);
}

int qs_single_query_attention_quant(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                    const int64_t* kv_pointers, const int32_t* length_per_sample, int8_t* out_q, void* out_scale, void* out_sum, int batch,
                                    int num_heads, int num_kv_heads, int head_dim, int max_blocks_per_seq, int memory_max_seqlen, int tokens_per_block,
                                    int size_per_token, int timestep, int rotary_embedding_dim, float rotary_base, int int4_kv_cache,
                                    int kv_cache_with_zeros, void* workspace, size_t workspace_bytes, void* stream) {
  QS_REQUIRE(q && k && v && kv_pointers && out_q && out_scale, "single_query_attention_quant: null tensor");
  DecodeAttnArgs a;
  a.q = q; a.k = k; a.v = v; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
  a.kv_pointers = reinterpret_cast<const long long*>(kv_pointers); a.lengths = length_per_sample; a.out = nullptr;
  a.q_out = out_q; a.q_scale = out_scale; a.q_sum = out_sum; a.workspace = workspace; a.workspace_bytes = workspace_bytes; a.prof = g_gemm_prof;
  a.batch = batch; a.num_heads = num_heads; a.num_kv_heads = num_kv_heads; a.head_dim = head_dim; a.max_blocks = max_blocks_per_seq;
  a.tokens_per_block = tokens_per_block; a.size_per_token = size_per_token; a.timestep = timestep; a.memory_max_len = memory_max_seqlen;
  a.rotary_dim = rotary_embedding_dim; a.rotary_base = rotary_base; a.int4_kv = int4_kv_cache; a.kv_zeros = kv_cache_with_zeros;
  a.stream = stream;
  return decode_attention(a);
}

int qs_apply_bias_rope_update_kv_cache(void* qkv, const int32_t* seq_lens, const int32_t* padding_offset, const int64_t* kv_pointers, int batch,
                                       int num_tokens, int max_blocks_per_seq, int head_num, int kv_head_num, int head_dim, int seq_len,
                                       int tokens_per_block, int size_per_token, int rotary_embedding_dim, float rotary_embedding_base,
                                       int rotary_embedding_max_positions, int neox_rotary_style, int int4_kv_cache, int kv_cache_with_zeros,
                                       void* stream) {
  (void)neox_rotary_style;
  QS_REQUIRE(qkv && seq_lens, "apply_bias_rope_update_kv_cache: null tensor");
  PrefillAppendArgs a;
  a.qkv = qkv; a.seq_lens = seq_lens; a.padding_offset = padding_offset; a.kv_pointers = reinterpret_cast<const long long*>(kv_pointers);
  a.batch = batch; a.num_tokens = num_tokens; a.max_blocks = max_blocks_per_seq; a.num_heads = head_num; a.num_kv_heads = kv_head_num;
  a.head_dim = head_dim; a.seq_len = seq_len; a.tokens_per_block = tokens_per_block; a.size_per_token = size_per_token;
  a.rotary_dim = rotary_embedding_dim; a.rotary_base = rotary_embedding_base; a.max_positions = rotary_embedding_max_positions;
  a.int4_kv = int4_kv_cache; a.kv_zeros = kv_cache_with_zeros; a.stream = stream;
  return prefill_rope_append(a);
}

// what every operator over portions in the paged cache asks of its arguments
static int paged_cache(PagedCache& c, const char* op, const int64_t* kv_pointers, const int32_t* cu_seqlens, const int32_t* lengths, int batch, int num_tokens,
                       int max_blocks, int num_kv_heads, int head_dim, int tokens_per_block, int size_per_token, int int4, int zeros) {
  QS_REQUIRE(batch >= 0 && num_tokens >= 0 && max_blocks >= 0, "%s: negative size", op);
  QS_REQUIRE(head_dim == 128, "%s: head_dim=%d, only 128 is supported", op, head_dim);
  QS_REQUIRE(zeros, "%s: only kv_cache_with_zeros=True is supported", op);
  QS_REQUIRE(tokens_per_block == 64, "%s: tokens_per_block=%d, only 64 is supported", op, tokens_per_block);
  QS_REQUIRE(num_kv_heads > 0 && size_per_token == static_cast<long long>(num_kv_heads) * 128 * (int4 ? 4 : 8) / 8,
             "%s: size_per_token=%d does not match %d kv heads x %d bits", op, size_per_token, num_kv_heads, int4 ? 4 : 8);
  QS_REQUIRE(max_blocks <= (1 << 24), "%s: %d pages per sequence", op, max_blocks);
  if (batch > 0 && num_tokens > 0) QS_REQUIRE(kv_pointers && lengths, "%s: null tensor", op);
  c.kv_pointers = reinterpret_cast<const long long*>(kv_pointers);
  c.cu_seqlens = cu_seqlens;
  c.lengths = lengths;
  c.max_blocks = max_blocks;
  c.num_kv_heads = num_kv_heads;
  c.int4 = int4 != 0;
  return qs::QS_OK;
}
static int paged_rows(const char* op, const char* name, const void* t, int64_t stride, int heads) {
  QS_REQUIRE(t != nullptr, "%s: %s is null", op, name);
  QS_REQUIRE(aligned16(t) && stride % 8 == 0, "%s: rows of %s must start on 16-byte boundaries", op, name);
  QS_REQUIRE(stride >= static_cast<int64_t>(heads) * 128, "%s: row stride of %s smaller than the row", op, name);
  return qs::QS_OK;
}

static int append(AppendArgs& a, const char* op, const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride, void* q_out,
                  int64_t q_out_stride, const int64_t* kv_pointers, const int32_t* cu_seqlens, const int32_t* lengths, int batch, int num_tokens, int max_blocks_per_seq,
                  int num_heads, int num_kv_heads, int head_dim, int tokens_per_block, int size_per_token, int rotary_embedding_dim, float rotary_base,
                  int int4_kv_cache, int kv_cache_with_zeros, void* stream) {
  int rc = paged_cache(a.cache, op, kv_pointers, cu_seqlens, lengths, batch, num_tokens, max_blocks_per_seq, num_kv_heads, head_dim, tokens_per_block, size_per_token,
                       int4_kv_cache, kv_cache_with_zeros);
  if (rc) return rc;
  QS_REQUIRE(num_heads > 0 && num_heads % num_kv_heads == 0, "%s: heads %d / kv heads %d", op, num_heads, num_kv_heads);
  QS_REQUIRE(rotary_embedding_dim == head_dim, "%s: rotary_embedding_dim=%d must equal head_dim", op, rotary_embedding_dim);
  QS_REQUIRE(rotary_base > 0.f && rotary_base < 3.0e38f, "%s: rotary_base must be positive and finite", op);
  if (batch == 0 || num_tokens == 0) return qs::QS_OK;
  if ((rc = paged_rows(op, "q", q, q_stride, num_heads)) || (rc = paged_rows(op, "k", k, k_stride, num_kv_heads)) ||
      (rc = paged_rows(op, "v", v, v_stride, num_kv_heads)) || (rc = paged_rows(op, "out", q_out, q_out_stride, num_heads)))
    return rc;
  a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.q_out_stride = q_out_stride;
  a.batch = batch; a.num_tokens = num_tokens; a.num_heads = num_heads; a.rotary_base = rotary_base; a.stream = stream;
  return append_kv_cache(a);
}

int qs_append_kv_cache(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride, void* q_out, int64_t q_out_stride,
                       const int64_t* kv_pointers, const int32_t* cu_seqlens, const int32_t* lengths, int batch, int num_tokens, int max_blocks_per_seq,
                       int num_heads, int num_kv_heads, int head_dim, int tokens_per_block, int size_per_token, int rotary_embedding_dim, float rotary_base,
                       int int4_kv_cache, int kv_cache_with_zeros, void* stream) {
  AppendArgs a;
  return append(a, "append_kv_cache", q, k, v, q_stride, k_stride, v_stride, q_out, q_out_stride, kv_pointers, cu_seqlens, lengths, batch, num_tokens, max_blocks_per_seq,
                num_heads, num_kv_heads, head_dim, tokens_per_block, size_per_token, rotary_embedding_dim, rotary_base, int4_kv_cache, kv_cache_with_zeros, stream);
}

int qs_append_kv_cache_at(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride, void* q_out, int64_t q_out_stride,
                          const int64_t* kv_pointers, const int32_t* cu_seqlens, const int32_t* lengths, const int32_t* positions, const int32_t* rotary_sections,
                          int axes, int interleaved, int batch, int num_tokens, int max_blocks_per_seq, int num_heads, int num_kv_heads, int head_dim, int tokens_per_block,
                          int size_per_token, int rotary_embedding_dim, float rotary_base, int int4_kv_cache, int kv_cache_with_zeros, void* stream) {
  const char* op = "append_kv_cache_at";
  QS_REQUIRE(axes >= 1 && axes <= 4, "%s: %d axes, 1 to 4 are supported", op, axes);
  QS_REQUIRE(rotary_sections != nullptr, "%s: rotary_sections is null", op);
  int sum = 0;
  for (int i = 0; i < axes; ++i) {
    QS_REQUIRE(rotary_sections[i] >= 0 && rotary_sections[i] <= 64, "%s: a rotary section of %d pairs", op, rotary_sections[i]);
    sum += rotary_sections[i];
  }
  QS_REQUIRE(sum == 64, "%s: rotary sections of %d pairs in all, a head has 64", op, sum);
  AppendArgs a;
  if (interleaved) {  // pair i is of axis i mod axes as long as that has pairs left, then of the first
    for (int i = 0; i < 64; ++i) a.axis_of[i] = static_cast<unsigned char>(i % axes > 0 && i / axes < rotary_sections[i % axes] ? i % axes : 0);
    for (int i = 1; i < axes; ++i)
      QS_REQUIRE(rotary_sections[i] <= (64 - i + axes - 1) / axes, "%s: %d interleaved pairs of axis %d of %d", op, rotary_sections[i], i, axes);
  } else {
    int axis = 0, end = rotary_sections[0];
    for (int i = 0; i < 64; ++i) {
      while (i >= end) end += rotary_sections[++axis];
      a.axis_of[i] = static_cast<unsigned char>(axis);
    }
  }
  if (batch > 0 && num_tokens > 0) QS_REQUIRE(positions != nullptr, "%s: positions is null", op);
  a.positions = positions;
  return append(a, op, q, k, v, q_stride, k_stride, v_stride, q_out, q_out_stride, kv_pointers, cu_seqlens, lengths, batch, num_tokens, max_blocks_per_seq, num_heads,
                num_kv_heads, head_dim, tokens_per_block, size_per_token, rotary_embedding_dim, rotary_base, int4_kv_cache, kv_cache_with_zeros, stream);
}

int qs_keep_kv_cache(int32_t* new_lengths, const int64_t* kv_pointers, const int32_t* cu_seqlens, const int32_t* lengths, const int32_t* rows, const int32_t* counts,
                     int max_rows, int batch, int num_tokens, int max_blocks_per_seq, int num_kv_heads, int head_dim, int tokens_per_block, int size_per_token,
                     int int4_kv_cache, int kv_cache_with_zeros, void* stream) {
  const char* op = "keep_kv_cache";
  PagedCache c;
  const int rc = paged_cache(c, op, kv_pointers, cu_seqlens, lengths, batch, num_tokens, max_blocks_per_seq, num_kv_heads, head_dim, tokens_per_block, size_per_token,
                             int4_kv_cache, kv_cache_with_zeros);
  if (rc) return rc;
  QS_REQUIRE(max_rows >= 0 && max_rows <= kMostDrafted, "%s: %d rows of a portion, at most %d are supported", op, max_rows, kMostDrafted);
  QS_REQUIRE(batch <= 65535, "%s: batch=%d exceeds the grid limits", op, batch);
  if (batch == 0) return qs::QS_OK;
  QS_REQUIRE(new_lengths && lengths && counts && (rows || max_rows == 0), "%s: null tensor", op);
  QS_REQUIRE(new_lengths != lengths, "%s: the new lengths must have a place of their own", op);
  QS_REQUIRE(kv_pointers || max_blocks_per_seq == 0, "%s: null tensor", op);
  return keep_kv_cache(new_lengths, c, rows, counts, max_rows, batch, num_tokens, stream);
}

int qs_read_kv_cache(void* k_out, void* v_out, const int64_t* kv_pointers, const int32_t* cu_seqlens, const int32_t* lengths, int batch, int num_tokens,
                     int max_blocks_per_seq, int num_kv_heads, int head_dim, int tokens_per_block, int size_per_token, int int4_kv_cache, int kv_cache_with_zeros,
                     void* stream) {
  const char* op = "read_kv_cache";
  PagedCache c;
  int rc = paged_cache(c, op, kv_pointers, cu_seqlens, lengths, batch, num_tokens, max_blocks_per_seq, num_kv_heads, head_dim, tokens_per_block, size_per_token,
                       int4_kv_cache, kv_cache_with_zeros);
  if (rc || batch == 0 || num_tokens == 0) return rc;
  if ((rc = paged_rows(op, "k", k_out, num_kv_heads * 128, num_kv_heads)) || (rc = paged_rows(op, "v", v_out, num_kv_heads * 128, num_kv_heads))) return rc;
  return read_kv_cache(k_out, v_out, c, batch, num_tokens, stream);
}

size_t qs_paged_prompt_attention_workspace_bytes(int batch, int num_tokens, int max_seqlen, int max_length, int num_heads, int num_kv_heads) {
  return paged_prompt_workspace(batch, num_tokens, max_seqlen, max_length, num_heads, num_kv_heads);
}

static int prompt_attention(PagedAttnArgs& a, const char* op, const void* q, int64_t q_stride, void* out, int64_t out_stride, const int64_t* kv_pointers,
                            const int32_t* cu_seqlens, const int32_t* lengths, int batch, int num_tokens, int max_seqlen, int max_length, int max_blocks_per_seq, int num_heads,
                            int num_kv_heads, int head_dim, int tokens_per_block, int size_per_token, int int4_kv_cache, int kv_cache_with_zeros, float softmax_scale,
                            void* workspace, size_t workspace_bytes, void* stream) {
  int rc = paged_cache(a.cache, op, kv_pointers, cu_seqlens, lengths, batch, num_tokens, max_blocks_per_seq, num_kv_heads, head_dim, tokens_per_block, size_per_token,
                       int4_kv_cache, kv_cache_with_zeros);
  if (rc) return rc;
  QS_REQUIRE(num_heads > 0 && num_heads % num_kv_heads == 0, "%s: heads %d / kv heads %d", op, num_heads, num_kv_heads);
  QS_REQUIRE(max_seqlen >= 0 && max_length >= 0, "%s: negative size", op);
  QS_REQUIRE(softmax_scale > 0.f && softmax_scale < 1.0e30f, "%s: softmax_scale must be positive and finite", op);
  if (batch == 0 || num_tokens == 0 || max_seqlen == 0) return qs::QS_OK;
  if ((rc = paged_rows(op, "q", q, q_stride, num_heads)) || (rc = paged_rows(op, "out", out, out_stride, num_heads))) return rc;
  QS_REQUIRE(aligned16(workspace), "%s: workspace must be 16-byte aligned", op);
  a.q = q; a.out = out; a.q_stride = q_stride; a.out_stride = out_stride; a.batch = batch; a.num_tokens = num_tokens; a.num_heads = num_heads;
  a.max_seqlen = max_seqlen < num_tokens ? max_seqlen : num_tokens; a.max_length = max_length; a.softmax_scale = softmax_scale;
  a.workspace = workspace; a.workspace_bytes = workspace_bytes; a.stream = stream;
  return paged_prompt_attention(a);
}

int qs_paged_prompt_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride, const int64_t* kv_pointers, const int32_t* cu_seqlens,
                              const int32_t* lengths, int batch, int num_tokens, int max_seqlen, int max_length, int max_blocks_per_seq, int num_heads,
                              int num_kv_heads, int head_dim, int tokens_per_block, int size_per_token, int int4_kv_cache, int kv_cache_with_zeros,
                              float softmax_scale, void* workspace, size_t workspace_bytes, void* stream) {
  PagedAttnArgs a;
  return prompt_attention(a, "paged_prompt_attention", q, q_stride, out, out_stride, kv_pointers, cu_seqlens, lengths, batch, num_tokens, max_seqlen, max_length,
                          max_blocks_per_seq, num_heads, num_kv_heads, head_dim, tokens_per_block, size_per_token, int4_kv_cache, kv_cache_with_zeros, softmax_scale, workspace,
                          workspace_bytes, stream);
}

size_t qs_paged_tree_attention_workspace_bytes(int batch, int num_tokens, int max_seqlen, int max_length, int num_heads, int num_kv_heads) {
  return paged_tree_workspace(batch, num_tokens, max_seqlen, max_length, num_heads, num_kv_heads);
}

int qs_paged_tree_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride, const int64_t* kv_pointers, const int32_t* cu_seqlens,
                            const int32_t* lengths, const int64_t* visible, int visible_words, int batch, int num_tokens, int max_seqlen, int max_length,
                            int max_blocks_per_seq, int num_heads, int num_kv_heads, int head_dim, int tokens_per_block, int size_per_token, int int4_kv_cache,
                            int kv_cache_with_zeros, float softmax_scale, void* workspace, size_t workspace_bytes, void* stream) {
  const char* op = "paged_tree_attention";
  PagedAttnArgs a;
  if (batch > 0 && num_tokens > 0 && max_seqlen > 0) {
    QS_REQUIRE(visible != nullptr && (reinterpret_cast<uintptr_t>(visible) & 7) == 0, "%s: visible must be there, on an 8-byte boundary", op);
    QS_REQUIRE(visible_words > 0 && visible_words <= (1 << 24) && static_cast<long long>(visible_words) * 64 >= (max_seqlen < num_tokens ? max_seqlen : num_tokens),
               "%s: %d words of 64 rows for portions of %d", op, visible_words, max_seqlen);
  }
  a.visible = reinterpret_cast<const unsigned long long*>(visible);
  a.visible_words = visible_words;
  return prompt_attention(a, op, q, q_stride, out, out_stride, kv_pointers, cu_seqlens, lengths, batch, num_tokens, max_seqlen, max_length,
                          max_blocks_per_seq, num_heads, num_kv_heads, head_dim, tokens_per_block, size_per_token, int4_kv_cache, kv_cache_with_zeros, softmax_scale, workspace,
                          workspace_bytes, stream);
}

int qs_draft_tree(int32_t* positions, int64_t* visible, const int32_t* parents, const int32_t* cu_seqlens, const int32_t* lengths, int batch, int num_tokens, int max_seqlen,
                  void* stream) {
  QS_REQUIRE(batch >= 0 && num_tokens >= 0, "draft_tree: negative size");
  QS_REQUIRE(max_seqlen >= 0 && max_seqlen <= kMostDrafted, "draft_tree: max_seqlen=%d, at most %d rows of a portion are supported", max_seqlen, kMostDrafted);
  if (batch == 0 || num_tokens == 0 || max_seqlen == 0) return qs::QS_OK;
  QS_REQUIRE(positions && visible && parents && lengths, "draft_tree: null tensor");
  return draft_tree(positions, reinterpret_cast<long long*>(visible), parents, cu_seqlens, lengths, batch, num_tokens, max_seqlen, stream);
}

int qs_verify_drafts(int64_t* out_tokens, int32_t* out_rows, int32_t* out_counts, const void* logits, int logits_type, int64_t logits_stride, const int64_t* tokens,
                     const int32_t* parents, const float* draft_probs, int64_t probs_stride, const int32_t* cu_seqlens, const float* coins, const float* draws,
                     const float* temperatures, int batch, int num_tokens, int vocab, int max_seqlen, void* stream) {
  const char* op = "verify_drafts";
  QS_REQUIRE(batch >= 0 && num_tokens >= 0, "%s: negative size", op);
  QS_REQUIRE(max_seqlen >= 0 && max_seqlen <= kMostDrafted, "%s: max_seqlen=%d, at most %d rows of a portion are supported", op, max_seqlen, kMostDrafted);
  QS_REQUIRE(logits_type >= 0 && logits_type <= 2, "%s: logits of type %d", op, logits_type);
  QS_REQUIRE(vocab > 0 && vocab <= (1 << 28), "%s: vocab=%d", op, vocab);
  QS_REQUIRE(batch <= (1 << 24), "%s: %d sequences", op, batch);
  QS_REQUIRE(!(parents && draft_probs), "%s: draft probabilities go with chains, not with parents", op);
  if (batch == 0) return qs::QS_OK;
  QS_REQUIRE(out_counts && ((out_tokens && out_rows) || max_seqlen == 0), "%s: null tensor", op);
  if (num_tokens > 0) {
    QS_REQUIRE(logits && tokens && coins && draws, "%s: null tensor", op);
    QS_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (logits_type == 2 ? 3 : 1)) == 0, "%s: logits must start on a boundary of their type", op);
    QS_REQUIRE(num_tokens == 1 || logits_stride >= vocab, "%s: row stride of logits smaller than the row", op);
    QS_REQUIRE((reinterpret_cast<uintptr_t>(draft_probs) & 3) == 0, "%s: draft_probs must start on a boundary of its type", op);
    QS_REQUIRE(!draft_probs || num_tokens == 1 || probs_stride >= vocab, "%s: row stride of draft_probs smaller than the row", op);
  }
  VerifyArgs a;
  a.logits = logits; a.type = logits_type; a.logits_stride = logits_stride; a.probs_stride = probs_stride; a.tokens = reinterpret_cast<const long long*>(tokens);
  a.parents = parents; a.probs = draft_probs; a.cu_seqlens = cu_seqlens; a.coins = coins; a.draws = draws; a.temperatures = temperatures;
  a.out_tokens = reinterpret_cast<long long*>(out_tokens); a.out_rows = out_rows; a.out_counts = out_counts; a.batch = batch; a.num_tokens = num_tokens; a.vocab = vocab;
  a.max_seqlen = max_seqlen; a.stream = stream;
  return verify_drafts(a);
}

size_t qs_shared_prefix_attention_workspace_bytes(int batch, int shared_blocks, int num_heads, int num_kv_heads) {
  return shared_prefix_workspace(batch, shared_blocks, num_heads, num_kv_heads);
}

int qs_shared_prefix_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride, const int64_t* kv_pointers, const int32_t* lengths, int batch,
                               int shared_blocks, int max_length, int max_blocks_per_seq, int num_heads, int num_kv_heads, int head_dim, int tokens_per_block,
                               int size_per_token, int int4_kv_cache, int kv_cache_with_zeros, float softmax_scale, void* workspace, size_t workspace_bytes,
                               void* stream) {
  const char* op = "shared_prefix_attention";
  PagedAttnArgs a;
  int rc = paged_cache(a.cache, op, kv_pointers, nullptr, lengths, batch, batch, max_blocks_per_seq, num_kv_heads, head_dim, tokens_per_block, size_per_token,
                       int4_kv_cache, kv_cache_with_zeros);
  if (rc) return rc;
  QS_REQUIRE(num_heads > 0 && num_heads % num_kv_heads == 0, "%s: heads %d / kv heads %d", op, num_heads, num_kv_heads);
  QS_REQUIRE(shared_blocks >= 0 && shared_blocks <= max_blocks_per_seq, "%s: shared_blocks=%d of %d pages per sequence", op, shared_blocks, max_blocks_per_seq);
  QS_REQUIRE(max_length >= 0, "%s: negative size", op);
  QS_REQUIRE(softmax_scale > 0.f && softmax_scale < 1.0e30f, "%s: softmax_scale must be positive and finite", op);
  QS_REQUIRE(batch <= 65535 && num_heads <= 65535, "%s: batch=%d / heads=%d exceed the grid limits", op, batch, num_heads);
  if (batch == 0) return qs::QS_OK;
  if ((rc = paged_rows(op, "q", q, q_stride, num_heads)) || (rc = paged_rows(op, "out", out, out_stride, num_heads))) return rc;
  QS_REQUIRE(aligned16(workspace), "%s: workspace must be 16-byte aligned", op);
  a.q = q; a.out = out; a.q_stride = q_stride; a.out_stride = out_stride; a.batch = batch; a.num_tokens = batch; a.num_heads = num_heads; a.max_seqlen = 1;
  a.max_length = max_length; a.softmax_scale = softmax_scale; a.workspace = workspace; a.workspace_bytes = workspace_bytes; a.stream = stream;
  return shared_prefix_attention(a, shared_blocks);
}

int qs_prefill_attention(const void* q, const void* k, const void* v, int64_t q_stride, int64_t k_stride, int64_t v_stride, void* out,
                         int64_t out_stride, const int32_t* cu_seqlens, int batch, int num_tokens, int max_seqlen, int num_heads, int num_kv_heads,
                         int head_dim, float softmax_scale, void* stream) {
  PrefillAttnArgs a;
  a.q = q; a.k = k; a.v = v; a.out = out; a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.out_stride = out_stride;
  a.cu_seqlens = cu_seqlens; a.batch = batch; a.num_tokens = num_tokens; a.max_seqlen = max_seqlen; a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads; a.head_dim = head_dim; a.softmax_scale = softmax_scale; a.stream = stream;
  return prefill_attention(a);
}

int qs_compute_padding_offsets(int32_t* out, const int32_t* cu_seqlens, int batch, int max_seqlen, void* stream) {
  QS_REQUIRE(out && cu_seqlens, "compute_padding_offsets: null tensor");
  return padding_offsets(out, cu_seqlens, batch, max_seqlen, stream);
}

int qs_rms_norm(void* out, const void* input, const void* weight, float epsilon, int use_quant, int tokens, int hidden, void* stream) {
  QS_REQUIRE(out && input && weight, "rms_norm: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(input) && aligned16(weight), "rms_norm: tensors must be 16-byte aligned");
  return rms_norm(out, input, weight, epsilon, use_quant, tokens, hidden, stream);
}

int qs_rms_norm_general(int8_t* out, const void* input, const void* weight, void* scaling, float epsilon, int use_per_token_quant, int tokens,
                        int hidden, void* stream) {
  QS_REQUIRE(out && input && weight && scaling, "rms_norm_general: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(input) && aligned16(weight), "rms_norm_general: tensors must be 16-byte aligned");
  return layernorm_general_quant(out, input, weight, nullptr, scaling, epsilon, tokens, hidden, use_per_token_quant, stream);
}

int qs_rms_norm_general_fuse_sum(int8_t* out, const void* input, const void* weight, void* input_sum, void* scaling, float epsilon,
                                 int use_per_token_quant, int tokens, int hidden, void* stream) {
  QS_REQUIRE(out && input && weight && scaling && input_sum, "rms_norm_general_fuse_sum: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(input) && aligned16(weight), "rms_norm_general_fuse_sum: tensors must be 16-byte aligned");
  return layernorm_general_quant(out, input, weight, input_sum, scaling, epsilon, tokens, hidden, use_per_token_quant, stream);
}

int qs_dequant_add_residual_rms_norm_quant(int8_t* out, const int32_t* input, void* residual, const void* gamma, const void* scale_vec,
                                           float scale, float epsilon, int tokens, int hidden, void* stream) {
  QS_REQUIRE(out && input && residual && gamma, "invoke_dequant_add_residual_rms_norm_quant: null tensor");
  return dequant_add_residual_rms_norm_quant(out, input, residual, gamma, scale_vec, scale, epsilon, tokens, hidden, stream);
}

int qs_invoke_quant(int8_t* out, const void* input, void* scale, int tokens, int hidden, void* stream) {
  QS_REQUIRE(out && input && scale, "invoke_quant: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(input), "invoke_quant: tensors must be 16-byte aligned");
  return quant_per_token(out, input, nullptr, scale, tokens, hidden, stream);
}
int qs_invoke_quant_scalar(int8_t* out, const void* input, float scale, int tokens, int hidden, void* stream) {
  QS_REQUIRE(out && input, "invoke_quant: null tensor");
  return quant_scalar(out, input, scale, tokens, hidden, stream);
}
int qs_invoke_quant_fuse_sum(int8_t* out, const void* input, void* input_sum, void* scale, int tokens, int hidden, void* stream) {
  QS_REQUIRE(out && input && scale && input_sum, "invoke_quant_fuse_sum: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(input), "invoke_quant_fuse_sum: tensors must be 16-byte aligned");
  return quant_per_token(out, input, input_sum, scale, tokens, hidden, stream);
}
int qs_add_rms_norm_general_peer(int8_t* out, void* hidden_out, const void* x, const void* const* delta_ptrs, void* const* flag_ptrs, void* state, int world,
                                 int rank, int phase, const void* gamma, void* input_sum, void* scaling, float epsilon, int tokens, int hidden, void* stream) {
  QS_REQUIRE(out && hidden_out && x && delta_ptrs && flag_ptrs && state && gamma && scaling, "add_rms_norm_general_peer: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(hidden_out) && aligned16(x) && aligned16(gamma), "add_rms_norm_general_peer: tensors must be 16-byte aligned");
  return add_layernorm_quant_peer(out, hidden_out, x, delta_ptrs, flag_ptrs, state, world, rank, phase, gamma, input_sum, scaling, epsilon, tokens, hidden, stream);
}
int qs_row_absmax(float* amax_out, const void* input, int tokens, int hidden, void* stream) {
  QS_REQUIRE(amax_out && input, "row_absmax: null tensor");
  QS_REQUIRE(aligned16(input), "row_absmax: input must be 16-byte aligned");
  return row_absmax(amax_out, input, tokens, hidden, stream);
}
int qs_invoke_quant_given_amax(int8_t* out, const void* input, const float* amax, void* input_sum, void* scale, int tokens, int hidden, void* stream) {
  QS_REQUIRE(out && input && amax && scale, "invoke_quant_given_amax: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(input), "invoke_quant_given_amax: tensors must be 16-byte aligned");
  return quant_given_amax(out, input, amax, input_sum, scale, tokens, hidden, stream);
}
int qs_invoke_dequant_add_residual(void* out, const int32_t* input, const void* residual, const void* scale_vec, float scale, int tokens,
                                   int hidden, void* stream) {
  QS_REQUIRE(out && input && residual, "invoke_dequant_add_residual: null tensor");
  return dequant_add_residual(out, input, residual, scale_vec, scale, tokens, hidden, stream);
}
int qs_invoke_dequant(void* out, const int32_t* input, float scale, int tokens, int hidden, int input_stride, int out_stride, void* stream) {
  QS_REQUIRE(out && input, "invoke_dequant: null tensor");
  return dequant(out, input, scale, tokens, hidden, input_stride, out_stride, stream);
}

int qs_argmax_rows(int64_t* out, const void* logits, int rows, int vocab, void* stream) {
  QS_REQUIRE(out && logits, "argmax_rows: null tensor");
  QS_REQUIRE(aligned16(logits) && (static_cast<size_t>(vocab) * 2) % 16 == 0, "argmax_rows: rows must be 16-byte aligned");
  return argmax_rows(out, logits, rows, vocab, stream);
}

int qs_silu_and_mul_quant(int8_t* out, const void* input, void* input_sum, void* scale, int tokens, int d, void* stream) {
  QS_REQUIRE(out && input && scale, "silu_and_mul_quant: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(input), "silu_and_mul_quant: tensors must be 16-byte aligned");
  return silu_and_mul_quant(out, input, input_sum, scale, tokens, d, stream);
}
int qs_add_rms_norm_general(int8_t* out, void* hidden_out, const void* x, const void* delta, const void* weight, void* input_sum, void* scaling,
                            float epsilon, int tokens, int hidden, void* stream) {
  QS_REQUIRE(out && hidden_out && x && delta && weight && scaling, "add_rms_norm_general: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(hidden_out) && aligned16(x) && aligned16(delta) && aligned16(weight), "add_rms_norm_general: tensors must be 16-byte aligned");
  return add_layernorm_quant(out, hidden_out, x, delta, weight, input_sum, scaling, epsilon, tokens, hidden, stream);
}
int qs_silu_and_mul(void* out, const void* input, int tokens, int d, void* stream) {
  QS_REQUIRE(out && input, "silu_and_mul: null tensor");
  QS_REQUIRE(aligned16(out) && aligned16(input), "silu_and_mul: tensors must be 16-byte aligned");
  return silu_and_mul(out, input, tokens, d, stream);
}
int qs_gelu_new(void* out, const void* input, int tokens, int d, void* stream) {
  QS_REQUIRE(out && input, "gelu_new: null tensor");
  return gelu(out, input, tokens, d, 0, stream);
}
int qs_gelu_fast(void* out, const void* input, int tokens, int d, void* stream) {
  QS_REQUIRE(out && input, "gelu_fast: null tensor");
  return gelu(out, input, tokens, d, 1, stream);
}
int qs_dequant_silu_and_mul_quant(int8_t* out, const int32_t* input, float scale_gate, float scale_up, float scale_out, float* scale_out_vec,
                                  float* tmp, int tokens, int d, void* stream) {
  QS_REQUIRE(out && input, "invoke_dequant_silu_and_mul_quant: null tensor");
  QS_REQUIRE((scale_out_vec == nullptr) == (tmp == nullptr), "invoke_dequant_silu_and_mul_quant: scale_out and tmp must be given together");
  return dequant_silu_and_mul_quant(out, input, scale_gate, scale_up, scale_out, scale_out_vec, tmp, tokens, d, stream);
}

}  // extern "C"
