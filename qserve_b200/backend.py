"""Host-side mirror of the reference's `qserve_backend` operator API on top of the C ABI.

Every public function has the name, positional argument order, argument meaning, ownership rules and error
behaviour (RuntimeError) of the pybind11 function it replaces (reference file:line in each docstring), so that
`qserve/modeling/layers/*` and `qserve/modeling/models/llama_w4a8_unpad.py` run unchanged against it.
PyTorch is used only for what the reference uses it for at this boundary: tensor metadata, the current CUDA
stream and the two outputs the reference ops allocate themselves.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import check, lib
from . import _bind  # after the library it links against

_HALF = torch.float16


# --------------------------------------------------------------------------------------------------
# plumbing
# --------------------------------------------------------------------------------------------------


def _call(t: torch.Tensor, fn, *args) -> None:
    """Launch `fn(*args, stream)` on the current stream of t's device, with that device current (the reference ops hold an
    at::cuda::CUDAGuard on the input's device, fused_attention.cpp:203); raises RuntimeError on failure."""
    idx = t.device.index
    cur = torch.cuda.current_device()
    if idx is None or idx == cur:
        check(fn(*args, torch._C._cuda_getCurrentRawStream(cur)))
    else:
        with torch.cuda.device(idx):
            check(fn(*args, torch._C._cuda_getCurrentRawStream(idx)))


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _cuda(t: torch.Tensor, name: str) -> None:
    _require(t.is_cuda, f"{name} must be on CUDA")  # CHECK_DEVICE, fused_attention.cpp:22


def _index(device: torch.device) -> int:
    return torch.cuda.current_device() if device.index is None else device.index


def gemm_workspace(device: torch.device) -> torch.Tensor:
    """Zero-initialised once per device; afterwards owned by the library (self-cleaning split-K counters)."""
    return _bind.gemm_workspace(_index(device))


def attention_workspace(device: torch.device, batch: int, num_heads: int, head_dim: int) -> torch.Tensor:
    """Grown on demand; a work space that was handed out is never freed: a captured CUDA graph may still hold its address (the self-cleaning
    counters inside must not alias reused memory on replay)."""
    return _bind.attention_workspace(_index(device), batch, num_heads, head_dim)


def set_pdl(enabled: bool) -> bool:
    """Toggle programmatic dependent launch for all subsequently launched kernels; returns the previous setting."""
    return bool(lib.qs_set_pdl(1 if enabled else 0))


# --------------------------------------------------------------------------------------------------
# qgemm_w4a8_per_chn / qgemm_w4a8_per_group / qgemm_w8a8
# --------------------------------------------------------------------------------------------------


def w4a8_per_chn_gemm_forward_cuda(in_feats, kernel, wscales, ascales, w_szs, a_ssums, out_feats, _acc_out=None) -> None:
    """qserve_backend.qgemm_w4a8_per_chn.gemm_forward_cuda (w4a8_per_chn/gemm_cuda.cu:596-652, pybind.cpp:13-16).

    out_feats[M,N] (fp16, caller allocated) = (in_feats s8 [M,K] . kernel u4 [N,K/2]) * wscales[n] * ascales[m] - w_szs[n] * a_ssums[m].
    """
    _bind.w4a8_per_chn(in_feats, kernel, wscales, ascales, w_szs, a_ssums, out_feats, _acc_out)


def w4a8_per_group_gemm_forward_cuda(in_feats, kernel, zeros, scales_i8, wscales, ascales, out_feats, _acc_out=None) -> None:
    """qserve_backend.qgemm_w4a8_per_group.gemm_forward_cuda (w4a8_per_group/gemm_cuda.cu:630-702).

    Argument order as called by w4a8_linear.py:123-131: (x, qweight, s2_zeros, s2_scales, s1_scales, input_scales, out).
    """
    _bind.w4a8_per_group(in_feats, kernel, zeros, scales_i8, wscales, ascales, out_feats, _acc_out)


def w8a8_gemm_forward_cuda(in_feats, kernel, wscales, ascales, out_feats, _acc_out=None) -> None:
    """qserve_backend.qgemm_w8a8.w8a8_gemm_forward_cuda (w8a8/w8a8_gemm_cuda.cu:532-577, pybind.cpp:13-17)."""
    _bind.w8a8(in_feats, kernel, wscales, ascales, out_feats, _acc_out)


# --------------------------------------------------------------------------------------------------
# fused_attention
# --------------------------------------------------------------------------------------------------


def single_query_attention(q, k, v, kv_pointers, length_per_sample_: Optional[torch.Tensor], alibi_slopes_: Optional[torch.Tensor],
                           memory_max_seqlen: int, tokens_per_block: int, size_per_token: int, timestep: int,
                           rotary_embedding_dim: int, rotary_base: float, neox_rotary_style: bool, int4_kv_cache: bool,
                           kv_cache_with_zeros: bool) -> torch.Tensor:
    """qserve_backend.fused_attention.single_query_attention (fused_attention.cpp:150-240).

    Returns a NEW tensor shaped like q (the reference returns torch::empty_like(q), :205).  Mutates the KV pages.
    """
    return _bind.single_query_attention(q, k, v, kv_pointers, length_per_sample_, alibi_slopes_, memory_max_seqlen, tokens_per_block, size_per_token, timestep,
                                        rotary_embedding_dim, rotary_base, neox_rotary_style, int4_kv_cache, kv_cache_with_zeros)


def apply_bias_rope_update_kv_cache(qkv, seq_lens, padding_offset, kv_pointers: Optional[torch.Tensor], head_num: int, kv_head_num: int,
                                    seq_len: int, tokens_per_block: int, size_per_token: int, rotary_embedding_dim: int,
                                    rotary_embedding_base: float, rotary_embedding_max_positions: int, neox_rotary_style: bool,
                                    int4_kv_cache: bool, kv_cache_with_zeros: bool) -> None:
    """qserve_backend.fused_attention.apply_bias_rope_update_kv_cache (update_kv_cache.cu:20-108): in-place RoPE on the
    packed qkv [T,(Hq+2Hkv)*D] and per-token-per-head asymmetric quantisation of K/V into the pages."""
    _cuda(qkv, "qkv")
    _require(qkv.dtype == _HALF and qkv.is_contiguous(), "qkv must be contiguous float16")
    _require(seq_lens.dtype == torch.int32 and padding_offset.dtype == torch.int32, "seq_lens and padding_offset must be int32")
    head_dim = int(rotary_embedding_dim)  # size_per_head = rotary_embedding_dim (update_kv_cache.cu:54)
    _require(qkv.size(-1) == (head_num + 2 * kv_head_num) * head_dim, "qkv width does not match (head_num + 2*kv_head_num) * head_dim")
    kvp, max_blocks = None, 0
    if kv_pointers is not None:
        _require(kv_pointers.is_contiguous() and kv_pointers.dtype == torch.int64, "kv_pointers must be contiguous int64")
        kvp, max_blocks = kv_pointers.data_ptr(), kv_pointers.size(-1)
    _call(qkv, _bind.qs_apply_bias_rope_update_kv_cache, qkv.data_ptr(), seq_lens.data_ptr(), padding_offset.data_ptr(), kvp, seq_lens.size(0), qkv.size(0),
                                                 max_blocks, int(head_num), int(kv_head_num), head_dim, int(seq_len), int(tokens_per_block),
                                                 int(size_per_token), int(rotary_embedding_dim), float(rotary_embedding_base),
                                                 int(rotary_embedding_max_positions), int(bool(neox_rotary_style)), int(bool(int4_kv_cache)),
                                                 int(bool(kv_cache_with_zeros)))


def compute_padding_offsets(cu_seqlens, max_seqlen: int, tot_num_tokens: int) -> torch.Tensor:
    """qserve_backend.fused_attention.compute_padding_offsets (input_metadata_helper.cu:33-45): returns int32 [tot_num_tokens]."""
    _cuda(cu_seqlens, "cu_seqlens")
    _require(cu_seqlens.dtype == torch.int32, "cu_seqlens must be int32")
    out = torch.empty((tot_num_tokens,), dtype=torch.int32, device=cu_seqlens.device)
    _call(cu_seqlens, _bind.qs_compute_padding_offsets, out.data_ptr(), cu_seqlens.data_ptr(), cu_seqlens.size(0) - 1, int(max_seqlen))
    return out


def flash_attn_varlen_func(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q: int, max_seqlen_k: int, dropout_p: float = 0.0,
                           softmax_scale: Optional[float] = None, causal: bool = False, **unsupported) -> torch.Tensor:
    """Drop-in for the ONE way the reference calls flash_attn.flash_attn_varlen_func (llama_w4a8_unpad.py:232-242): causal self-attention over a
    batch of prompts, q [T,Hq,128], k / v [T,Hkv,128] fp16 (strided views of the rotated qkv buffer are fine), the same cu_seqlens for queries
    and keys, no dropout.  Returns fp16 [T,Hq,128].  Anything else raises: this is not a general flash-attention."""
    _cuda(q, "q")
    _require(not unsupported or all(val in (None, False, 0, 0.0, (-1, -1)) for val in unsupported.values()), f"unsupported arguments {sorted(unsupported)}")
    _require(causal and float(dropout_p) == 0.0, "only causal=True, dropout_p=0.0 is implemented")
    _require(q.dtype == _HALF and k.dtype == _HALF and v.dtype == _HALF, "q, k, v must be float16")
    _require(q.dim() == 3 and k.dim() == 3 and v.dim() == 3 and q.size(2) == 128 and k.size(2) == 128 and v.size(2) == 128, "q, k, v must be [T, H, 128]")
    _require(k.shape == v.shape and q.size(0) == k.size(0), "q, k, v must cover the same tokens; k and v the same heads")
    _require(cu_seqlens_q.dtype == torch.int32 and cu_seqlens_q.is_contiguous(), "cu_seqlens must be contiguous int32")
    _require(cu_seqlens_k is cu_seqlens_q or (cu_seqlens_k.shape == cu_seqlens_q.shape and cu_seqlens_k.data_ptr() == cu_seqlens_q.data_ptr())
             or bool(torch.equal(cu_seqlens_k, cu_seqlens_q)), "queries and keys must share cu_seqlens (prompt self-attention)")
    _require(int(max_seqlen_q) == int(max_seqlen_k), "max_seqlen_q and max_seqlen_k must agree")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _require(t.stride(2) == 1 and t.stride(1) == 128, f"{name}: heads must be contiguous rows of 128 halfs")
    T, hq, hkv = q.size(0), q.size(1), k.size(1)
    out = torch.empty((T, hq, 128), dtype=_HALF, device=q.device)
    if T == 0:
        return out
    scale = float(softmax_scale) if softmax_scale is not None else 128 ** -0.5
    _call(q, _bind.qs_prefill_attention, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), k.stride(0), v.stride(0), out.data_ptr(), out.stride(0),
          cu_seqlens_q.data_ptr(), cu_seqlens_q.size(0) - 1, T, int(max_seqlen_q), hq, hkv, 128, scale)
    return out


# --------------------------------------------------------------------------------------------------
# layernorm_ops
# --------------------------------------------------------------------------------------------------


def _rows(t: torch.Tensor):
    hidden = t.size(-1)
    return (t.numel() // hidden if hidden else 0), hidden


def _noop(t: torch.Tensor) -> bool:
    """Empty batches are a no-op (the reference launches a zero-sized grid); data_ptr() of an empty tensor is NULL."""
    return t.numel() == 0


def _half_only(t: torch.Tensor, op: str) -> None:
    _require(t.dtype == _HALF, f"{op}: only float16 activations are supported by qserve_b200 (models run .half(), model_runner.py:148)")


def rms_norm(out, input, weight, epsilon: float, use_quant: bool = False) -> None:
    """layernorm_ops.rms_norm (layernorm.cpp:48-50, layernorm_kernels.cu:404-425)."""
    _cuda(input, "input"); _half_only(input, "rms_norm")
    if _noop(input):
        return
    tokens, hidden = _rows(input)
    _call(input, lib.qs_rms_norm, out.data_ptr(), input.data_ptr(), weight.data_ptr(), float(epsilon), int(bool(use_quant)), tokens, hidden)


def rms_norm_general(out, input, weight, scaling, epsilon: float, use_per_token_quant: bool = False) -> None:
    """layernorm_ops.rms_norm_general (layernorm.cpp:52-54, layernorm_kernels.cu:427-464)."""
    _bind.rms_norm_general(out, input, weight, scaling, epsilon, use_per_token_quant)


def rms_norm_general_fuse_sum(out, input, weight, input_sum, scaling, epsilon: float, use_per_token_quant: bool = False) -> None:
    """layernorm_ops.rms_norm_general_fuse_sum (layernorm.cpp:56-58, layernorm_kernels.cu:466-508)."""
    _bind.rms_norm_general_fuse_sum(out, input, weight, input_sum, scaling, epsilon, use_per_token_quant)


def invoke_dequant_add_residual_rms_norm_quant(out, input, residual, gamma, scale, epsilon: float) -> None:
    """layernorm_ops.invoke_dequant_add_residual_rms_norm_quant, scalar-Half and Tensor scale overloads (layernorm.cpp:60-71)."""
    _cuda(input, "input"); _half_only(residual, "invoke_dequant_add_residual_rms_norm_quant")
    if _noop(input):
        return
    tokens, hidden = _rows(input)
    if isinstance(scale, torch.Tensor):
        _call(input, lib.qs_dequant_add_residual_rms_norm_quant, out.data_ptr(), input.data_ptr(), residual.data_ptr(), gamma.data_ptr(), scale.data_ptr(), 0.0,
                                                         float(epsilon), tokens, hidden)
    else:
        s = float(torch.tensor(float(scale), dtype=_HALF))  # at::Half argument
        _call(input, lib.qs_dequant_add_residual_rms_norm_quant, out.data_ptr(), input.data_ptr(), residual.data_ptr(), gamma.data_ptr(), None, s,
                                                         float(epsilon), tokens, hidden)


# --------------------------------------------------------------------------------------------------
# fused_kernels
# --------------------------------------------------------------------------------------------------


def invoke_quant(out, input, scale) -> None:
    """fused_kernels.invoke_quant: Tensor scale [tokens] (written) or scalar Half scale (read)  (fused.cpp:52-58)."""
    if isinstance(scale, torch.Tensor):
        _bind.invoke_quant(out, input, scale)
        return
    _cuda(input, "input"); _half_only(input, "invoke_quant")
    _require(input.is_contiguous() and out.is_contiguous(), "invoke_quant: input and out must be contiguous")  # asserts, fused_kernels.cu:202-203
    if _noop(input):
        return
    tokens, hidden = _rows(input)
    s = float(torch.tensor(float(scale), dtype=_HALF))
    _call(input, lib.qs_invoke_quant_scalar, out.data_ptr(), input.data_ptr(), s, tokens, hidden)


def invoke_quant_fuse_sum(out, input, input_sum, scale) -> None:
    """fused_kernels.invoke_quant_fuse_sum (fused.cpp:59-69, fused_kernels.cu:234-265)."""
    if isinstance(scale, torch.Tensor):
        _bind.invoke_quant_fuse_sum(out, input, input_sum, scale)
        return
    _cuda(input, "input"); _half_only(input, "invoke_quant_fuse_sum")
    _require(input.is_contiguous() and out.is_contiguous(), "invoke_quant_fuse_sum: input and out must be contiguous")
    if _noop(input):
        return
    tokens, hidden = _rows(input)
    # scalar overload: static scale, the sum argument is unused by the reference kernel (fused_kernels.cu:131-136)
    s = float(torch.tensor(float(scale), dtype=_HALF))
    _call(input, lib.qs_invoke_quant_scalar, out.data_ptr(), input.data_ptr(), s, tokens, hidden)


def invoke_dequant_add_residual(out, input, residual, scale) -> None:
    """fused_kernels.invoke_dequant_add_residual, both overloads (fused.cpp:48-55)."""
    _cuda(input, "input"); _half_only(residual, "invoke_dequant_add_residual")
    if _noop(input):
        return
    tokens, hidden = _rows(input)
    if isinstance(scale, torch.Tensor):
        _call(input, lib.qs_invoke_dequant_add_residual, out.data_ptr(), input.data_ptr(), residual.data_ptr(), scale.data_ptr(), 0.0, tokens, hidden)
    else:
        s = float(torch.tensor(float(scale), dtype=_HALF))
        _call(input, lib.qs_invoke_dequant_add_residual, out.data_ptr(), input.data_ptr(), residual.data_ptr(), None, s, tokens, hidden)


def invoke_dequant(out, input, scale) -> None:
    """fused_kernels.invoke_dequant (fused.cpp:56, fused_kernels.cu:179-196)."""
    _cuda(input, "input"); _half_only(out, "invoke_dequant")
    if _noop(input):
        return
    tokens, hidden = _rows(input)
    s = float(torch.tensor(float(scale), dtype=_HALF))
    _call(input, lib.qs_invoke_dequant, out.data_ptr(), input.data_ptr(), s, tokens, hidden, input.stride(-2), out.stride(-2))


# --------------------------------------------------------------------------------------------------
# activation_ops
# --------------------------------------------------------------------------------------------------


def silu_and_mul(out, input) -> None:
    """activation_ops.silu_and_mul (activation.cpp:26, activation_kernels.cu:84-97): out[..., d] = silu(x[..., :d]) * x[..., d:]."""
    _bind.silu_and_mul(out, input)


def gelu_new(out, input) -> None:
    """activation_ops.gelu_new (activation.cpp:27)."""
    _cuda(input, "input"); _half_only(input, "gelu_new")
    tokens, d = _rows(input)
    _call(input, lib.qs_gelu_new, out.data_ptr(), input.data_ptr(), tokens, d)


def gelu_fast(out, input) -> None:
    """activation_ops.gelu_fast (activation.cpp:28)."""
    _cuda(input, "input"); _half_only(input, "gelu_fast")
    tokens, d = _rows(input)
    _call(input, lib.qs_gelu_fast, out.data_ptr(), input.data_ptr(), tokens, d)


def invoke_dequant_silu_and_mul_quant(out, input, scale_gate: float, scale_up: float, scale_out, tmp: Optional[torch.Tensor] = None) -> None:
    """activation_ops.invoke_dequant_silu_and_mul_quant, scalar and per-token overloads (activation.cpp:29-38)."""
    _cuda(input, "input")
    d = input.size(-1) // 2
    tokens = input.numel() // input.size(-1) if input.size(-1) else 0
    if isinstance(scale_out, torch.Tensor):
        _require(tmp is not None, "per-token overload needs the tmp buffer")
        _call(input, lib.qs_dequant_silu_and_mul_quant, out.data_ptr(), input.data_ptr(), float(scale_gate), float(scale_up), 0.0, scale_out.data_ptr(),
                                                tmp.data_ptr(), tokens, d)
    else:
        _call(input, lib.qs_dequant_silu_and_mul_quant, out.data_ptr(), input.data_ptr(), float(scale_gate), float(scale_up), float(scale_out), None, None,
                                                tokens, d)


# --------------------------------------------------------------------------------------------------
# fused extensions (not part of the reference surface; bit-identical to the op sequences they replace)
# --------------------------------------------------------------------------------------------------


def add_rms_norm_general(out, hidden_out, x, delta, weight, input_sum: Optional[torch.Tensor], scaling, epsilon: float) -> None:
    """hidden_out = x + delta (fp16, as torch computes `residual + out_buf`), then rms_norm_general[_fuse_sum](out, hidden_out, ...)."""
    _bind.add_rms_norm_general(out, hidden_out, x, delta, weight, input_sum, scaling, epsilon)


def silu_and_mul_quant(out, input, input_sum: Optional[torch.Tensor], scale) -> None:
    """silu_and_mul(input) followed by invoke_quant[_fuse_sum]; the fp16 activation never leaves the SM."""
    _bind.silu_and_mul_quant(out, input, input_sum, scale)


def single_query_attention_quant(q, k, v, kv_pointers, length_per_sample, memory_max_seqlen: int, tokens_per_block: int, size_per_token: int,
                                 timestep: int, rotary_embedding_dim: int, rotary_base: float, int4_kv_cache: bool, kv_cache_with_zeros: bool,
                                 out_q, out_scale, out_sum: Optional[torch.Tensor]) -> None:
    """single_query_attention + invoke_quant[_fuse_sum] in one launch: out_q int8 [B, Hq*D], out_scale / out_sum fp16 [B].
    Bit-identical to the two reference ops run back to back (llama_w4a8_unpad.py:265-283)."""
    _bind.single_query_attention_quant(q, k, v, kv_pointers, length_per_sample, memory_max_seqlen, tokens_per_block, size_per_token, timestep,
                                       rotary_embedding_dim, rotary_base, int4_kv_cache, kv_cache_with_zeros, out_q, out_scale, out_sum)


# --------------------------------------------------------------------------------------------------
# portions of sequences in the paged cache (extensions: the reference appends whole prompts only, and attends over keys of the same call)
#
# A flat batch of rows holds the last cu_seqlens[b + 1] - cu_seqlens[b] positions of sequence b (cu_seqlens int32 [B + 1]; None: one row per sequence);
# lengths int32 [B] counts what the sequence's pages hold with them, kv_pointers int64 [B, 2, blocks] as for single_query_attention, pages 16-byte aligned.
# Heads are 128 wide and contiguous, rows start on 16-byte boundaries.  Rows behind the last sequence (a padded batch) are not written:
# those of a given `out` stay as they are, those of a new result are unset.
# --------------------------------------------------------------------------------------------------


def append_kv_cache(q, k, v, kv_pointers, cu_seqlens: Optional[torch.Tensor], lengths, tokens_per_block: int, size_per_token: int, rotary_embedding_dim: int,
                    rotary_base: float, int4_kv_cache: bool, kv_cache_with_zeros: bool, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """RoPE of q [T,Hq,128] and k [T,Hkv,128] at the rows' positions, per-token-per-head quantisation of k and v into the pages: what
    apply_bias_rope_update_kv_cache does for whole prompts, for portions that continue sequences (single tokens among them).  Returns the rotated q (`out`
    may be q itself); q, k and v are not changed.  A row of equal values is held as that value; one that reaches the ends of fp16 reads
    as finite numbers, one with an infinity or NaN as NaN."""
    return _bind.append_kv_cache(q, k, v, kv_pointers, cu_seqlens, lengths, tokens_per_block, size_per_token, rotary_embedding_dim, rotary_base, int4_kv_cache,
                                 kv_cache_with_zeros, out)


def read_kv_cache(kv_pointers, cu_seqlens: Optional[torch.Tensor], lengths, num_tokens: int, tokens_per_block: int, size_per_token: int, int4_kv_cache: bool,
                  kv_cache_with_zeros: bool):
    """What the pages stand for at the last positions of the sequences: two new tensors k, v fp16 [num_tokens,Hkv,128] (num_tokens >= cu_seqlens[-1]).
    A whole sequence is read with cu_seqlens over its length.  Zeros for a row without a position in its sequence's pages."""
    return _bind.read_kv_cache(kv_pointers, cu_seqlens, lengths, num_tokens, tokens_per_block, size_per_token, int4_kv_cache, kv_cache_with_zeros)


def paged_prompt_attention(q, kv_pointers, cu_seqlens: Optional[torch.Tensor], lengths, max_seqlen: int, max_length: int, tokens_per_block: int,
                           size_per_token: int, int4_kv_cache: bool, kv_cache_with_zeros: bool, softmax_scale: Optional[float] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the rotated q [T,Hq,128] of portions over positions 0 .. its own of each row's sequence, keys and values out of the pages (those of the
    portion too: append_kv_cache first).  max_seqlen >= the longest portion, max_length >= the longest sequence.  Returns fp16 [T,Hq,128]; a row without a position
    (lengths[b] smaller than the portion) gets zeros.  softmax_scale > 0, default 128 ** -0.5."""
    return _bind.paged_prompt_attention(q, kv_pointers, cu_seqlens, lengths, max_seqlen, max_length, tokens_per_block, size_per_token, int4_kv_cache,
                                        kv_cache_with_zeros, softmax_scale, out)


def shared_prefix_attention(q, kv_pointers, lengths, shared_blocks: int, max_length: int, tokens_per_block: int, size_per_token: int, int4_kv_cache: bool,
                            kv_cache_with_zeros: bool, softmax_scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one rotated row per sequence, q [B,Hq,128], over its lengths[b] positions, all out of the pages (the new token's too: append_kv_cache first),
    where the first `shared_blocks` pages of all sequences are the same pages (they are taken from kv_pointers[0], whatever the other rows hold there): those are read
    and unpacked once for the whole batch.  A sequence may end within the shared pages; lengths[b] = 0 gets zeros.  max_length >= the longest sequence."""
    return _bind.shared_prefix_attention(q, kv_pointers, lengths, shared_blocks, max_length, tokens_per_block, size_per_token, int4_kv_cache, kv_cache_with_zeros,
                                         softmax_scale, out)


# --------------------------------------------------------------------------------------------------
# steps of several drafted tokens, and tokens with places of their own (extensions)
#
# The rows of a portion as above: row 0 is the token that the step starts from, the others are drafted tokens, each with a parent among the rows ahead of it.  A step:
# draft_tree, then append_kv_cache_at and paged_tree_attention in every layer, verify_drafts, keep_kv_cache in every layer.  A chain needs no positions of its own and
# nothing kept: append_kv_cache; what was not accepted lies behind the new lengths, lengths - portion + counts, and is written over.  Its attention is
# paged_prompt_attention, or paged_tree_attention with draft_tree's visible of parents -1, 0, 1, ..: the same numbers to their roundings, sooner where sequences have few
# rows (4 rows of 32 heads over 8, INT4: 18 sequences behind 3000 28 us in place of 53, 64 of them 87 for 135, 4 behind 60000 99 for 208).
# --------------------------------------------------------------------------------------------------


def draft_tree(parents, cu_seqlens: Optional[torch.Tensor], lengths, max_seqlen: int):
    """What the rows of drafted trees see of their portions, and where they are rotated: parents int32 [T] are rows within the portion, ahead of their children (row
    0's is not looked at).  Returns positions int32 [T] (the portion's first position + depth) and visible int64 [T, ceil(max_seqlen / 64)], bit i of a row: row i is the
    row itself or an ancestor.  A row whose parent does not lie ahead of it (-1) is padding and sees nothing of its portion.  max_seqlen <= 256."""
    return _bind.draft_tree(parents, cu_seqlens, lengths, max_seqlen)


def append_kv_cache_at(q, k, v, kv_pointers, cu_seqlens: Optional[torch.Tensor], lengths, positions, rotary_sections, tokens_per_block: int, size_per_token: int,
                       rotary_embedding_dim: int, rotary_base: float, int4_kv_cache: bool, kv_cache_with_zeros: bool, interleaved: bool = False,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """append_kv_cache with the angles given: positions int32 [T] (depths of a tree, with rotary_sections None or (64,)) or [axes, T] (time, height, width of images),
    where rotary_sections says how many of a head's 64 pairs go by each of one to four axes, one axis behind the other; interleaved: pair i goes by axis i mod axes as long
    as that one has pairs left, then by the first.  Where rows lie in the pages goes by lengths and cu_seqlens alone."""
    return _bind.append_kv_cache_at(q, k, v, kv_pointers, cu_seqlens, lengths, positions, rotary_sections, tokens_per_block, size_per_token, rotary_embedding_dim,
                                    rotary_base, int4_kv_cache, kv_cache_with_zeros, interleaved, out)


def paged_tree_attention(q, kv_pointers, cu_seqlens: Optional[torch.Tensor], lengths, visible, max_seqlen: int, max_length: int, tokens_per_block: int,
                         size_per_token: int, int4_kv_cache: bool, kv_cache_with_zeros: bool, softmax_scale: Optional[float] = None,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """paged_prompt_attention with what a row sees given: all positions ahead of its portion, and of the portion the rows whose bits it has in visible int64 [T, words]
    (bit i % 64 of word i / 64, 64 * words >= max_seqlen): a drafted tree's ancestors, an image that sees itself as a whole, several documents in one portion.  Its
    own place counts only by its bit, and later rows may be seen.  A row that sees nothing gets zeros.  Up to 16 rows a kv head (max_seqlen * heads / kv heads; not of
    few long sequences) and small calls take codes and weights as they are, and results are off by their own rounding, 2.1e-4; others hold keys, values and weights in
    fp16, as paged_prompt_attention does, 3.2e-4 to 4.8e-4: which of the two goes by the sizes of the whole call."""
    return _bind.paged_tree_attention(q, kv_pointers, cu_seqlens, lengths, visible, max_seqlen, max_length, tokens_per_block, size_per_token, int4_kv_cache,
                                      kv_cache_with_zeros, softmax_scale, out)


def verify_drafts(logits, draft_tokens, cu_seqlens: Optional[torch.Tensor], max_seqlen: int, coins, draws, parents: Optional[torch.Tensor] = None,
                  draft_probs: Optional[torch.Tensor] = None, temperatures: Optional[torch.Tensor] = None):
    """Which drafted tokens the target takes, and the token behind them, so that all are distributed as if drawn from the target one by one.  logits [T, vocab] fp16,
    bf16 or fp32, row i's behind row i; draft_tokens int64 [T] (row 0's is not looked at); coins fp32 [T] and draws fp32 [B] random in [0, 1); temperatures fp32 [B],
    0 or less: greedy, None: 1.  Drafts as they come, a chain or (with parents, as in draft_tree) a tree: of a row's children the first one at which the sum of their
    probabilities p exceeds the row's coin is taken, otherwise the sequence ends with a token drawn from the others.  Chains drawn at random from draft_probs fp32
    [T, vocab] (row i: what row i + 1's token was drawn from): a token x is taken where coin q(x) < p(x), otherwise the sequence ends with one drawn from max(p - q, 0).
    Returns tokens int64 [B, max_seqlen], rows int32 [B, max_seqlen] and counts int32 [B]: the rows taken, from row 0 on, the token behind each, and how many; -1 beyond.
    A row's child that is no token (outside the vocabulary) counts as one that was refused, so a chain that ends early ends its portion, or has zeros for q there.
    Logits of -inf or NaN are no tokens; a row with nothing else gives -1.  max_seqlen <= 256.  Decisions and draws are those of 64-bit sums, but for max(p - q, 0): tokens
    whose p and q differ by less than a 32-bit sum's error may count with up to that error, no more than 1e-4 of what is drawn from in all."""
    return _bind.verify_drafts(logits, draft_tokens, cu_seqlens, max_seqlen, coins, draws, parents, draft_probs, temperatures)


def keep_kv_cache(kv_pointers, cu_seqlens: Optional[torch.Tensor], lengths, rows, counts, tokens_per_block: int, size_per_token: int, int4_kv_cache: bool,
                  kv_cache_with_zeros: bool) -> torch.Tensor:
    """The rows that verify_drafts took, side by side at the front of their portions: position first + j gets what first + rows[b, j] holds, j < counts[b] (rows int32
    [B, <= 256], counts int32 [B]).  Returns the new lengths int32 [B], first + counts.  A row outside its portion (-1) leaves its place as it is."""
    return _bind.keep_kv_cache(kv_pointers, cu_seqlens, lengths, rows, counts, tokens_per_block, size_per_token, int4_kv_cache, kv_cache_with_zeros)


class PeerContext:
    """Peer-mapped buffers of a tensor-parallel group for the fused all-reduce (qs_add_rms_norm_general_peer): built once from
    torch.distributed._symmetric_memory (device memory + NVLink peer mappings are torch's plumbing; the kernel is ours).
    Layout of the symmetric allocation on every rank: [2 phases][tokens, hidden] fp16 partial outputs, then a 256-byte flag pad."""

    def __init__(self, tokens: int, hidden: int, device: torch.device, group):
        import ctypes

        import torch.distributed as dist
        import torch.distributed._symmetric_memory as symm

        self.world, self.rank = dist.get_world_size(group), dist.get_rank(group)
        _require(self.world <= 8, "PeerContext: at most 8 ranks")
        self.tokens, self.hidden = tokens, hidden
        phase_bytes = tokens * hidden * 2
        with torch.cuda.device(device):
            self.buf = symm.empty(2 * phase_bytes + 256, dtype=torch.uint8, device=device)
            self.buf.zero_()
            self.handle = symm.rendezvous(self.buf, group.group_name if hasattr(group, "group_name") else group)
            self.state = torch.zeros(4, dtype=torch.int32, device=device)
        torch.cuda.synchronize(device)
        dist.barrier(group)  # every rank's pad is zeroed before anyone signals
        base = [int(p) for p in self.handle.buffer_ptrs]
        self.partial = [self.buf[p * phase_bytes:(p + 1) * phase_bytes].view(torch.float16).view(tokens, hidden) for p in range(2)]  # local GEMM outputs
        arr = ctypes.c_void_p * self.world
        self._delta = [arr(*[b + p * phase_bytes for b in base]) for p in range(2)]
        self._flags = arr(*[b + 2 * phase_bytes for b in base])


def add_rms_norm_general_peer(out, hidden_out, x, ctx: "PeerContext", phase: int, weight, input_sum: Optional[torch.Tensor], scaling, epsilon: float) -> None:
    """add_rms_norm_general with delta = the sum over the tensor-parallel ranks of ctx.partial[phase] (fused all-reduce over peer memory)."""
    _cuda(x, "x"); _half_only(x, "add_rms_norm_general_peer")
    if _noop(x):
        return
    tokens, hidden = _rows(x)
    _require(tokens == ctx.tokens and hidden == ctx.hidden, "add_rms_norm_general_peer: shape does not match the PeerContext")
    _call(x, lib.qs_add_rms_norm_general_peer, out.data_ptr(), hidden_out.data_ptr(), x.data_ptr(), ctx._delta[phase], ctx._flags, ctx.state.data_ptr(),
          ctx.world, ctx.rank, int(phase), weight.data_ptr(), input_sum.data_ptr() if input_sum is not None else None, scaling.data_ptr(), float(epsilon),
          tokens, hidden)


def row_absmax(amax_out: torch.Tensor, input: torch.Tensor) -> None:
    """Tensor-parallel extension: amax_out[t] (fp32) = max |input[t, :]| of this rank's shard (then max-all-reduced by the caller)."""
    _cuda(input, "input"); _half_only(input, "row_absmax")
    _require(input.is_contiguous() and amax_out.dtype == torch.float32, "row_absmax: contiguous fp16 input, fp32 output")
    if _noop(input):
        return
    tokens, hidden = _rows(input)
    _call(input, lib.qs_row_absmax, amax_out.data_ptr(), input.data_ptr(), tokens, hidden)


def invoke_quant_given_amax(out, input, amax: torch.Tensor, input_sum: Optional[torch.Tensor], scale) -> None:
    """Tensor-parallel extension: invoke_quant[_fuse_sum] with a caller-supplied (global) per-token amax, fp32 [tokens]."""
    _cuda(input, "input"); _half_only(input, "invoke_quant_given_amax")
    _require(input.is_contiguous() and out.is_contiguous() and amax.dtype == torch.float32, "invoke_quant_given_amax: contiguous tensors, fp32 amax")
    if _noop(input):
        return
    tokens, hidden = _rows(input)
    _call(input, lib.qs_invoke_quant_given_amax, out.data_ptr(), input.data_ptr(), amax.data_ptr(), input_sum.data_ptr() if input_sum is not None else None,
          scale.data_ptr(), tokens, hidden)


def argmax_rows(logits: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """torch.argmax(logits, dim=-1) for fp16 logits [rows, vocab] in one launch (greedy sampling of the decode runner)."""
    _cuda(logits, "logits")
    _require(logits.dtype == _HALF and logits.dim() == 2 and logits.is_contiguous(), "logits must be contiguous float16 [rows, vocab]")
    if out is None:
        out = torch.empty(logits.size(0), dtype=torch.int64, device=logits.device)
    if logits.size(0) == 0:
        return out
    _call(logits, lib.qs_argmax_rows, out.data_ptr(), logits.data_ptr(), logits.size(0), logits.size(1))
    return out
