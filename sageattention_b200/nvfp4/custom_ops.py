"""`torch.library` registration of the NVFP4 operators, so that the path traces under
`torch.compile` / `torch.export` (fake-tensor shape inference) and takes part in autograd as
opaque ops.  The reference hints at this integration (`flash.py:268-273`) and upstream registers
its CUDA kernels the same way (`sageattention/sm80_compile.py:5-28, 98-132`).

Every op is a thin wrapper over the same host functions the eager API calls; nothing here adds a
second compute path.

    out = torch.ops.sageattention_b200.nvfp4_attn(q, k, v, scaling, causal, groups)     # differentiable
    nib, sc = torch.ops.sageattention_b200.nvfp4_quant(x, transpose, k_pad)
    out = torch.ops.sageattention_b200.nvfp4_decode(q, knv, ksc, vnv, vsc, s, s_pad, scaling, groups)
    out = nvfp4_attn_ex(q, k, v, scaling, causal, groups, key_pad_bias=..., cu_seqlens=..., out_layout=...,
                        backward_grad_dots=...)                                         # differentiable
    torch.ops.sageattention_b200.nvfp4_kv_append(k_new, v_new, knv, ksc, vnv, vsc, partial, rk, rv, pos)
    out = torch.ops.sageattention_b200.nvfp4_hybrid_decode(q, knv, ksc, vnv, vsc, rk, rv, length, window,
                                                           scaling, groups)
    slot_map, positions, cu, shortage = torch.ops.sageattention_b200.paged_kv_reserve(new, lengths, table, free, count, n, block)
    torch.ops.sageattention_b200.paged_kv_trim(keep, lengths, table, free, count, block)
    torch.ops.sageattention_b200.fp8_kv_write(key, value, slot_map, k_cache, v_cache, k_scale, v_scale)
    out, lse = torch.ops.sageattention_b200.fp8_paged_decode(q, k_cache, v_cache, k_scale, v_scale, table, lengths, scaling, groups)
    out, lse = torch.ops.sageattention_b200.fp8_paged_attention(q, cu, k_cache, v_cache, k_scale, v_scale, table, lengths,
                                                                scaling, groups)
    mask, positions = torch.ops.sageattention_b200.draft_tree(parents, cu, lengths, max_tokens)
    out, lse = torch.ops.sageattention_b200.fp8_paged_tree_attention(q, cu, mask, k_cache, v_cache, k_scale, v_scale, table,
                                                                     lengths, scaling, groups)
    accepted, num, following = torch.ops.sageattention_b200.verify_drafts(target_probs, tokens, parents, cu, uniforms, draft_probs,
                                                                                 max_tokens)
    keep = torch.ops.sageattention_b200.paged_kv_keep_path(accepted, num, cu, lengths, table, k_cache, v_cache, k_scale, v_scale)
    q, k = torch.ops.sageattention_b200.qk_norm_rope(q, k, wq, wk, cos, sin, positions, pos0, eps)       # differentiable
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import flash
from . import kv_cache as _kvc
from . import paged_cache as _paged

_NS = "sageattention_b200"


@torch.library.custom_op(f"{_NS}::nvfp4_attn_fwd", mutates_args=())
def nvfp4_attn_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scaling: float, causal: bool,
                   groups: int) -> Tuple[torch.Tensor, torch.Tensor]:
    out, lse = flash.nvfp4_flash_attention(q, k, v, scaling, causal=causal, num_key_value_groups=groups,
                                           return_lse=True)
    return out, lse


@nvfp4_attn_fwd.register_fake
def _(q, k, v, scaling, causal, groups):
    z, h, s_q, d = q.shape
    return q.new_empty(z, h, s_q, d), q.new_empty(z * h, s_q, dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::nvfp4_attn_bwd", mutates_args=())
def nvfp4_attn_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                   dout: torch.Tensor, scaling: float, causal: bool,
                   groups: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return flash._run_bwd_hp(q, k, v, out, lse, dout, scaling, causal, groups)


@nvfp4_attn_bwd.register_fake
def _(q, k, v, out, lse, dout, scaling, causal, groups):
    return (dout.new_empty(q.shape), dout.new_empty(k.shape), dout.new_empty(v.shape))


def _attn_setup(ctx, inputs, output):
    q, k, v, scaling, causal, groups = inputs
    out, lse = output
    ctx.save_for_backward(q, k, v, out, lse)
    ctx.meta = (scaling, causal, groups)


def _attn_backward(ctx, grad_out, grad_lse):
    q, k, v, out, lse = ctx.saved_tensors
    scaling, causal, groups = ctx.meta
    dq, dk, dv = nvfp4_attn_bwd(q, k, v, out, lse, grad_out.contiguous(), scaling, causal, groups)
    return dq, dk, dv, None, None, None


nvfp4_attn_fwd.register_autograd(_attn_backward, setup_context=_attn_setup)


def nvfp4_attn(q, k, v, scaling: float, causal: bool = False, groups: int = 1) -> torch.Tensor:
    """Differentiable attention through the registered ops (dense; `[Z,H,S,D]` layout)."""
    return nvfp4_attn_fwd(q, k, v, scaling, causal, groups)[0]


@torch.library.custom_op(f"{_NS}::nvfp4_quant", mutates_args=())
def nvfp4_quant(x: torch.Tensor, transpose: bool, k_pad: int) -> Tuple[torch.Tensor, torch.Tensor]:
    nib, sc = flash._quant_nvfp4(x, transpose=transpose, k_pad=k_pad if k_pad > 0 else None)
    return nib, sc.view(torch.uint8)


@nvfp4_quant.register_fake
def _(x, transpose, k_pad):
    b, a1, a2 = x.shape
    r, kk = (a2, a1) if transpose else (a1, a2)
    kp = k_pad if k_pad > 0 else kk
    return (x.new_empty(b, r, kp // 2, dtype=torch.uint8), x.new_empty(b, r, kp // 16, dtype=torch.uint8))


@torch.library.custom_op(f"{_NS}::nvfp4_decode", mutates_args=())
def nvfp4_decode(q: torch.Tensor, knv: torch.Tensor, ksc: torch.Tensor, vnv: torch.Tensor, vsc: torch.Tensor,
                 s: int, s_pad: int, scaling: float, groups: int) -> torch.Tensor:
    packed = (knv, ksc.view(torch.float8_e4m3fn), vnv, vsc.view(torch.float8_e4m3fn), s, s_pad)
    return flash.nvfp4_flash_decode_prequant(q, packed, scaling, groups)


@nvfp4_decode.register_fake
def _(q, knv, ksc, vnv, vsc, s, s_pad, scaling, groups):
    return q.new_empty(q.shape)


# ---------------------------------------------------------------- attention with every forward option
def _varlen(cu_seqlens, s_q, device):
    return flash._varlen_seq_arrays(cu_seqlens, s_q, device) if cu_seqlens is not None else None


@torch.library.custom_op(f"{_NS}::nvfp4_attn_ex_fwd", mutates_args=())
def nvfp4_attn_ex_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scaling: float, causal: bool,
                      groups: int, key_pad_bias: Optional[torch.Tensor], cu_seqlens: Optional[torch.Tensor],
                      out_zshd: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    out, lse = flash.nvfp4_flash_attention(
        q, k, v, scaling, causal=causal, num_key_value_groups=groups, key_pad_bias=key_pad_bias,
        return_lse=True, out_layout="zshd" if out_zshd else "zhsd", _varlen_arrays=_varlen(cu_seqlens, q.shape[2], q.device))
    return out, lse


@nvfp4_attn_ex_fwd.register_fake
def _(q, k, v, scaling, causal, groups, key_pad_bias, cu_seqlens, out_zshd):
    z, h, s_q, d = q.shape
    out = q.new_empty(z, s_q, h, d) if out_zshd else q.new_empty(z, h, s_q, d)
    return out, q.new_empty(z * h, s_q, dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::nvfp4_attn_ex_bwd", mutates_args=())
def nvfp4_attn_ex_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                      dout: torch.Tensor, scaling: float, causal: bool, groups: int,
                      key_pad_bias: Optional[torch.Tensor], cu_seqlens: Optional[torch.Tensor], out_zshd: bool,
                      grad_mode: str) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    varlen = _varlen(cu_seqlens, q.shape[2], q.device)
    layout = "zshd" if out_zshd else "zhsd"
    if grad_mode == "bf16":
        return flash._run_bwd_hp(q, k, v, out, lse, dout, scaling, causal, groups, varlen, layout,
                                 key_pad_bias=key_pad_bias)
    return flash._run_bwd(q, k, v, out, lse, dout, scaling, causal, groups, varlen, layout, mode=grad_mode,
                          key_pad_bias=key_pad_bias)


@nvfp4_attn_ex_bwd.register_fake
def _(q, k, v, out, lse, dout, scaling, causal, groups, key_pad_bias, cu_seqlens, out_zshd, grad_mode):
    return (dout.new_empty(q.shape), dout.new_empty(k.shape), dout.new_empty(v.shape))


class _AttnEx(torch.autograd.Function):
    """Autograd over the two registered ops (the backward mode is not an input of the forward op,
    so it travels on the context instead of through ``register_autograd``)."""

    @staticmethod
    def forward(ctx, q, k, v, scaling, causal, groups, key_pad_bias, cu_seqlens, out_zshd, grad_mode):
        out, lse = nvfp4_attn_ex_fwd(q, k, v, scaling, causal, groups, key_pad_bias, cu_seqlens, out_zshd)
        ctx.save_for_backward(q, k, v, out, lse, key_pad_bias, cu_seqlens)
        ctx.meta = (scaling, causal, groups, out_zshd, grad_mode)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        q, k, v, out, lse, bias, cu = ctx.saved_tensors
        scaling, causal, groups, out_zshd, grad_mode = ctx.meta
        dq, dk, dv = nvfp4_attn_ex_bwd(q, k, v, out, lse, grad_out, scaling, causal, groups, bias, cu, out_zshd,
                                       grad_mode)
        return (dq, dk, dv) + (None,) * 7


def nvfp4_attn_ex(q, k, v, scaling: float, causal: bool = False, groups: int = 1, key_pad_bias=None,
                  cu_seqlens=None, out_layout: str = "zhsd", backward_grad_dots: Optional[str] = None) -> torch.Tensor:
    """Differentiable attention through the registered ops with the options of
    ``nvfp4_flash_attn_func``: additive key bias, packed varlen rows (``cu_seqlens``), ``zshd``
    output, and the backward mode ("bf16", "fp4_rownorm", "fp4_legacy" without stochastic
    rounding, "fp8_rownorm"; None resolves like the eager entry)."""
    if out_layout not in ("zhsd", "zshd"):
        raise ValueError(f"out_layout must be 'zhsd' or 'zshd', got {out_layout!r}")
    s_kv = k.shape[2]
    eff = s_kv if cu_seqlens is None else q.shape[2] / max(1, cu_seqlens.numel() - 1)
    mode = flash._resolve_backward_grad_dots(backward_grad_dots, eff, False, groups)
    if cu_seqlens is not None:
        assert causal and q.shape[0] == 1 and q.shape[2] == s_kv, "varlen needs causal packed self-attention with Z == 1"
    return _AttnEx.apply(q, k, v, float(scaling), bool(causal), int(groups), key_pad_bias, cu_seqlens,
                         out_layout == "zshd", mode)


# ---------------------------------------------------------------- KV cache: append and hybrid decode
@torch.library.custom_op(f"{_NS}::nvfp4_kv_append",
                         mutates_args=("knv", "ksc", "vnv", "vsc", "v_partial", "rk", "rv"))
def nvfp4_kv_append(k_new: torch.Tensor, v_new: torch.Tensor, knv: torch.Tensor, ksc: torch.Tensor,
                    vnv: torch.Tensor, vsc: torch.Tensor, v_partial: torch.Tensor, rk: Optional[torch.Tensor],
                    rv: Optional[torch.Tensor], pos: int) -> None:
    """``NVFP4KVCache.append`` on the cache's buffers (scale tensors as float8_e4m3fn or uint8)."""
    _kvc.append_token(k_new, v_new, knv, ksc, vnv, vsc, v_partial, rk, rv, pos)


@nvfp4_kv_append.register_fake
def _(k_new, v_new, knv, ksc, vnv, vsc, v_partial, rk, rv, pos):
    return None


@torch.library.custom_op(f"{_NS}::nvfp4_hybrid_decode", mutates_args=())
def nvfp4_hybrid_decode(q: torch.Tensor, knv: torch.Tensor, ksc: torch.Tensor, vnv: torch.Tensor,
                        vsc: torch.Tensor, rk: torch.Tensor, rv: torch.Tensor, length: int, recent_window: int,
                        scaling: float, groups: int) -> torch.Tensor:
    """``NVFP4KVCache.hybrid_decode`` on the cache's buffers."""
    f8 = torch.float8_e4m3fn
    return _kvc.hybrid_decode_buffers(q, knv, ksc.view(f8) if ksc.dtype != f8 else ksc, vnv,
                                      vsc.view(f8) if vsc.dtype != f8 else vsc, rk, rv, length, recent_window,
                                      scaling, groups)


@nvfp4_hybrid_decode.register_fake
def _(q, knv, ksc, vnv, vsc, rk, rv, length, recent_window, scaling, groups):
    return q.new_empty(q.shape)


# ---------------------------------------------------------------- paged 8-bit KV cache
@torch.library.custom_op(f"{_NS}::paged_kv_reserve", mutates_args=("lengths", "block_table", "free_count"))
def paged_kv_reserve(new_lens: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, free_blocks: torch.Tensor,
                     free_count: torch.Tensor, num_slots: int,
                     block_size: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``paged_kv_reserve``: (slot_map, positions, cu_seqlens, shortage)."""
    return tuple(_paged.paged_kv_reserve(new_lens, lengths, block_table, free_blocks, free_count, num_slots, block_size))


@paged_kv_reserve.register_fake
def _(new_lens, lengths, block_table, free_blocks, free_count, num_slots, block_size):
    i32 = lambda n: new_lens.new_empty(n, dtype=torch.int32)
    return new_lens.new_empty(num_slots, dtype=torch.int64), i32(num_slots), i32(new_lens.shape[0] + 1), i32(1)


@torch.library.custom_op(f"{_NS}::paged_kv_trim", mutates_args=("lengths", "block_table", "free_blocks", "free_count"))
def paged_kv_trim(keep_lens: torch.Tensor, lengths: torch.Tensor, block_table: torch.Tensor, free_blocks: torch.Tensor,
                  free_count: torch.Tensor, block_size: int) -> None:
    _paged.paged_kv_trim(keep_lens, lengths, block_table, free_blocks, free_count, block_size)


@paged_kv_trim.register_fake
def _(keep_lens, lengths, block_table, free_blocks, free_count, block_size):
    return None


@torch.library.custom_op(f"{_NS}::fp8_kv_write", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def fp8_kv_write(key: torch.Tensor, value: torch.Tensor, slot_map: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
    """``fp8_kv_write`` (caches as float8_e4m3fn or uint8)."""
    _paged.fp8_kv_write(key, value, slot_map, k_cache, v_cache, k_scale, v_scale)


@fp8_kv_write.register_fake
def _(key, value, slot_map, k_cache, v_cache, k_scale, v_scale):
    return None


@torch.library.custom_op(f"{_NS}::fp8_paged_decode", mutates_args=())
def fp8_paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                     block_table: torch.Tensor, lengths: torch.Tensor, scaling: float,
                     groups: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return _paged.fp8_paged_decode(q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling, groups, return_lse=True)


@fp8_paged_decode.register_fake
def _(q, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling, groups):
    return q.new_empty(q.shape), q.new_empty(q.shape[0], q.shape[1], dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::fp8_paged_attention", mutates_args=())
def fp8_paged_attention(q: torch.Tensor, cu_seqlens: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, scaling: float,
                        groups: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return _paged.fp8_paged_attention(q, cu_seqlens, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling, groups,
                                      return_lse=True)


@fp8_paged_attention.register_fake
def _(q, cu_seqlens, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling, groups):
    return q.new_empty(q.shape), q.new_empty(q.shape[0], q.shape[1], dtype=torch.float32)


# ---------------------------------------------------------------- trees of drafts over the paged cache
@torch.library.custom_op(f"{_NS}::draft_tree", mutates_args=())
def draft_tree(parents: torch.Tensor, cu_seqlens: torch.Tensor, lengths: torch.Tensor, max_tokens: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """``draft_tree``: (tree_mask, positions)."""
    return tuple(_paged.draft_tree(parents, cu_seqlens, lengths, max_tokens))


@draft_tree.register_fake
def _(parents, cu_seqlens, lengths, max_tokens):
    t = parents.shape[0]
    return parents.new_empty(t, (max_tokens + 63) // 64, dtype=torch.int64), parents.new_empty(t, dtype=torch.int32)


@torch.library.custom_op(f"{_NS}::fp8_paged_tree_attention", mutates_args=())
def fp8_paged_tree_attention(q: torch.Tensor, cu_seqlens: torch.Tensor, tree_mask: torch.Tensor, k_cache: torch.Tensor,
                             v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
                             lengths: torch.Tensor, scaling: float, groups: int) -> Tuple[torch.Tensor, torch.Tensor]:
    return _paged.fp8_paged_tree_attention(q, cu_seqlens, tree_mask, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling,
                                           groups, return_lse=True)


@fp8_paged_tree_attention.register_fake
def _(q, cu_seqlens, tree_mask, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling, groups):
    return q.new_empty(q.shape), q.new_empty(q.shape[0], q.shape[1], dtype=torch.float32)


@torch.library.custom_op(f"{_NS}::verify_drafts", mutates_args=())
def verify_drafts(target_probs: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, cu_seqlens: torch.Tensor,
                  uniforms: torch.Tensor, draft_probs: Optional[torch.Tensor], max_tokens: int = 1024) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``verify_drafts``: (accepted, num_accepted, next_tokens)."""
    return tuple(_paged.verify_drafts(target_probs, tokens, parents, cu_seqlens, uniforms, draft_probs, max_tokens))


@verify_drafts.register_fake
def _(target_probs, tokens, parents, cu_seqlens, uniforms, draft_probs, max_tokens=1024):
    r = cu_seqlens.shape[0] - 1
    return (tokens.new_empty(tokens.shape[0], dtype=torch.int32), tokens.new_empty(r, dtype=torch.int32),
            tokens.new_empty(r, dtype=torch.int64))


@torch.library.custom_op(f"{_NS}::paged_kv_keep_path", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def paged_kv_keep_path(accepted: torch.Tensor, num_accepted: torch.Tensor, cu_seqlens: torch.Tensor, lengths: torch.Tensor,
                       block_table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                       v_scale: torch.Tensor) -> torch.Tensor:
    return _paged.paged_kv_keep_path(accepted, num_accepted, cu_seqlens, lengths, block_table, k_cache, v_cache, k_scale, v_scale)


@paged_kv_keep_path.register_fake
def _(accepted, num_accepted, cu_seqlens, lengths, block_table, k_cache, v_cache, k_scale, v_scale):
    return lengths.new_empty(lengths.shape)


# ---------------------------------------------------------------- norm of queries and keys with their rotation
def _rows_like(x):
    """As the operator lays results out: dense, heads inside or outside of tokens as in x."""
    if x.dim() == 4 and x.stride(1) < x.stride(2):
        z, h, s, d = x.shape
        return x.new_empty(z, s, h, d).transpose(1, 2)
    return x.new_empty(x.shape)


@torch.library.custom_op(f"{_NS}::qk_norm_rope", mutates_args=())
def qk_norm_rope(query: torch.Tensor, key: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, positions: Optional[torch.Tensor], pos0: int, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return flash.qk_norm_rope(query, key, q_weight, k_weight, cos, sin, positions, pos0, eps)


@qk_norm_rope.register_fake
def _(query, key, q_weight, k_weight, cos, sin, positions, pos0, eps):
    return _rows_like(query), _rows_like(key)


@torch.library.custom_op(f"{_NS}::qk_norm_rope_bwd", mutates_args=())
def qk_norm_rope_bwd(query: torch.Tensor, key: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                     sin: torch.Tensor, positions: Optional[torch.Tensor], pos0: int, eps: float, grad_q: torch.Tensor,
                     grad_k: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return flash._qk_norm_rope_backward(query, key, q_weight, k_weight, cos, sin, positions, pos0, eps, grad_q, grad_k)


@qk_norm_rope_bwd.register_fake
def _(query, key, q_weight, k_weight, cos, sin, positions, pos0, eps, grad_q, grad_k):
    return _rows_like(query), _rows_like(key), q_weight.new_empty(q_weight.shape), k_weight.new_empty(k_weight.shape)


def _norm_rope_setup(ctx, inputs, output):
    query, key, q_weight, k_weight, cos, sin, positions, pos0, eps = inputs
    ctx.save_for_backward(query, key, q_weight, k_weight, cos, sin, positions)
    ctx.meta = (pos0, eps)


def _norm_rope_backward(ctx, grad_q, grad_k):
    query, key, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
    grad_q = torch.zeros_like(query) if grad_q is None else grad_q
    grad_k = torch.zeros_like(key) if grad_k is None else grad_k
    return (*qk_norm_rope_bwd(query, key, q_weight, k_weight, cos, sin, positions, *ctx.meta, grad_q, grad_k), *[None] * 5)


qk_norm_rope.register_autograd(_norm_rope_backward, setup_context=_norm_rope_setup)
