"""Training-step operators around the attention, differentiable: rotary positions, activations kept in 8 bits for
the backward pass, and the next-token loss with its gradient in one pass.

  rotary_frequencies, apply_rotary     rotary positions on q and k, angles in 64 bits, half or interleaved pairs, all or
                                       part of the head, frequencies scaled for long contexts
                                       (RotaryEmbedding / apply_rotary_pos_emb, rope.py:11-185, cover half pairs over
                                       the whole head from 32-bit tables)
  pack_activation                      a tensor in 8 bits (PackedActivation)
  packed_add_rmsnorm, packed_silu_mul  the decoder layer's norm and SwiGLU product (gsa_llama.py:18-46) that keep
                                       their inputs in 8 bits; the backward pass differentiates at the kept values
  packed_mlp_block                     residual add, norm and MLP of a decoder layer (gsa_llama.py:100-110) as one
                                       node that keeps 1 + 2 d_ffn / d_model packed values per value of the stream
  fused_next_token_loss                GSALlamaForCausalLM's loss (gsa_llama.py:323-336)

The autograd functions are in csrc/torch_ops.cpp.  Each runs on its tensors' device and current stream and can be captured into a CUDA graph (a backward pass that is
captured must not share its leaves with a graph of eager operations that is still alive: torch binds the leaves'
accumulation to the stream of the first).  Second derivatives and forward-mode ones are not implemented, and refused.
"""

from __future__ import annotations

import math
from typing import Any, Dict, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .ops import PackedActivation


# ---------------------------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------------------------
def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[Dict[str, Any]] = None,
                       seq_len: Optional[int] = None, device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq [dim/2] fp64, attention factor) for apply_rotary, ``dim`` the rotated part of the head.

    ``scaling`` is a GSAConfig.rope_scaling dictionary; its "type" (or "rope_type") is one of

      none, "default"  base^(-2i/dim)
      "linear"         those / factor
      "ntk"            base * factor^(dim/(dim-2)) in place of base (rope.py:66-71)
      "dynamic_ntk"    the same with factor * seq_len / original_max_position_embeddings - (factor - 1) once seq_len
                       exceeds original_max_position_embeddings (the standard frequencies up to there)
      "yarn"           rope.py:73-101
      "llama3"         frequencies of wavelength over original / low_freq_factor divided by factor, those under
                       original / high_freq_factor kept, linear in original / wavelength between

    and its "attention_factor" (1 if absent, for "yarn" too) multiplies sines and cosines.

    The attention layer's own RotaryEmbedding gives the same angles for none, "ntk" and "yarn" under "type" only: any other
    type leaves it at the standard frequencies (rope.py:53-57), and it reads neither "rope_type" nor "attention_factor".
    Keys for a layer's cache are to be rotated with a dictionary that both read alike."""
    if dim < 2 or dim % 2:
        raise ValueError(f"rotary dim {dim} is not a positive even number")
    cfg = scaling or {}
    kind = cfg.get("type", cfg.get("rope_type"))
    factor = float(cfg.get("factor", 1.0))
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    f = float(base) ** (-i / dim)
    if kind in (None, "default"):
        pass
    elif kind == "linear":
        f = f / factor
    elif kind in ("ntk", "dynamic_ntk", "dynamic"):
        grow = factor
        if kind != "ntk":
            orig = int(cfg.get("original_max_position_embeddings", 4096))
            grow = factor * seq_len / orig - (factor - 1) if seq_len is not None and seq_len > orig else 1.0
        if dim > 2:  # a single frequency is 1 whatever the base
            f = (float(base) * grow ** (dim / (dim - 2))) ** (-i / dim)
    elif kind == "yarn":
        orig = cfg.get("original_max_position_embeddings", 4096)

        def pair_of(turns):  # the (fractional) pair that makes this many turns over the original context
            return dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(int(math.floor(pair_of(cfg.get("beta_fast", 32)))), 0)
        high = min(int(math.ceil(pair_of(cfg.get("beta_slow", 1)))), dim // 2 - 1)
        n = torch.arange(dim // 2, dtype=torch.float64)
        if high > low:
            stretch = ((n - low) / (high - low)).clamp(0.0, 1.0)
        else:
            stretch = (n >= low).double()
        f = f * (1 - stretch) + f / factor * stretch
    elif kind == "llama3":
        orig = float(cfg.get("original_max_position_embeddings", 8192))
        lo, hi = float(cfg.get("low_freq_factor", 1.0)), float(cfg.get("high_freq_factor", 4.0))
        if hi <= lo:
            raise ValueError(f"llama3 scaling: high_freq_factor {hi} <= low_freq_factor {lo}")
        keep = ((orig * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1 - keep)
    else:
        raise ValueError(f"unknown rope scaling type: {kind}")
    return f.to(device) if device is not None else f, float(cfg.get("attention_factor", 1.0))


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor,
                 attention_factor: float = 1.0, interleaved: bool = False, out=None):
    """(q', k'): q [B, L, H, D] and k [B, L, Hk, D] (or None) rotated to ``positions`` ([B, L], [1, L] or [L] integers)
    in the first ``2 * len(inv_freq)`` values of each head; the rest pass through.

    ``inv_freq`` and ``attention_factor`` come from rotary_frequencies and get no gradient (frequencies that want one are
    refused).  Pairs are (i, i + rotary_dim/2), or (2i, 2i+1) when ``interleaved``.  ``out=(q_out, k_out)`` (without
    autograd) receives the results: K straight into a cache's slots (``store.kv[:, n:n + L, 0]``), or the inputs themselves
    to rotate in place; outputs that overlap an input otherwise, or each other, are refused."""
    if torch.is_grad_enabled() and inv_freq.requires_grad:
        raise NotImplementedError("apply_rotary gives no gradient for inv_freq; detach it")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if out is not None:
            raise NotImplementedError("apply_rotary writes into given tensors without autograd only")
        return _lib.native().rotary_autograd(q, k, positions, inv_freq, attention_factor, interleaved)
    return ops.rotary(q, k, positions, inv_freq, attention_factor, interleaved, out=out)


# ---------------------------------------------------------------------------------------------
# Activations in 8 bits
# ---------------------------------------------------------------------------------------------
def pack_activation(x: torch.Tensor) -> PackedActivation:
    """x [..., n] in 8 bits (33/32 bytes a value); ``.unpack()`` gives it back."""
    return ops.pack_e4m3(x)


def packed_silu_mul(gu: torch.Tensor) -> torch.Tensor:
    """silu(g) * u of gu [..., 2n] = (g, u); the backward pass reads (g, u) from 8 bits."""
    if torch.is_grad_enabled() and gu.requires_grad:
        return _lib.native().silu_mul_autograd(gu)
    return ops.silu_mul_packed(gu)[0]


def packed_add_rmsnorm(x: torch.Tensor, a: Optional[torch.Tensor], weight: torch.Tensor, eps: float):
    """(h, y): h = x + a (x itself when a is None) and y = RMSNorm(h) * weight over the last dimension; the
    backward pass reads h from 8 bits."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, a, weight)):
        h, y = _lib.native().add_rmsnorm_autograd(x, a, weight, eps)
    else:
        h, y, _, _ = ops.add_rmsnorm_packed(x, a, weight, eps)
    return (x if a is None else h), y


class _PackedMlpBlock(torch.autograd.Function):
    """h = x + a, out = h + down(silu(gate(y)) * up(y)), y = RMSNorm(h) * weight.  Kept: h and (g, u) in 8 bits and
    the row statistics; y and silu(g) * u are formed again, by the kernels that run over the packed tensors
    anyway, for the weight gradients.  Everything is computed in the tensors' type, autocast or not: its products in another
    type would return the residual stream in that type, or meet kernels that take one type alone."""

    @staticmethod
    def forward(ctx, x, a, weight, w_gate, w_up, w_down, eps):
        d = x.shape[-1]
        h, y, ph, rstd = ops.add_rmsnorm_packed(x, a, weight, eps)
        h2 = (x if h is None else h).reshape(-1, d)
        y2 = y.view(-1, d)
        n = w_gate.shape[0]
        gu = torch.empty(y2.shape[0], 2 * n, device=x.device, dtype=x.dtype)
        with torch.autocast("cuda", enabled=False):
            torch.mm(y2, w_gate.t(), out=gu[:, :n])
            torch.mm(y2, w_up.t(), out=gu[:, n:])
            z, pgu = ops.silu_mul_packed(gu)
            out = torch.addmm(h2, z, w_down.t()).view(x.shape)
        ctx.save_for_backward(ph.data, rstd, pgu.data, weight, w_gate, w_up, w_down)
        ctx.forms = (ph.shape, ph.dtype), (pgu.shape, pgu.dtype)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        ph, rstd, pgu, weight, w_gate, w_up, w_down = ctx.saved_tensors
        form_h, form_gu = ctx.forms
        need = ctx.needs_input_grad
        d, n = w_gate.shape[1], w_gate.shape[0]
        do2 = d_out.reshape(-1, d)
        with torch.autocast("cuda", enabled=False):
            dgu, z = ops.silu_mul_packed_backward(do2 @ w_down, PackedActivation(pgu, *form_gu), want_z=need[5])
            d_down = do2.t() @ z if need[5] else None
            dg, du = dgu[:, :n], dgu[:, n:]
            dy = torch.addmm(dg @ w_gate, du, w_up)
            dx, dw, y = ops.rmsnorm_packed_backward(dy.view(d_out.shape), PackedActivation(ph, *form_h), rstd, weight,
                                                    dh=d_out, want_y=need[3] or need[4], want_dw=need[2])
            y2 = None if y is None else y.view(-1, d)
            return (dx if need[0] else None, dx if need[1] else None, dw, dg.t() @ y2 if need[3] else None,
                    du.t() @ y2 if need[4] else None, d_down, None)


def packed_mlp_block(x: torch.Tensor, a: Optional[torch.Tensor], weight: torch.Tensor, w_gate: torch.Tensor,
                     w_up: torch.Tensor, w_down: torch.Tensor, eps: float) -> torch.Tensor:
    """h + down(silu(gate(y)) * up(y)) with h = x + a (x when a is None) and y = RMSNorm(h) * weight: the second half of
    a pre-norm decoder layer, keeping its activations in 8 bits for the backward pass.  Tensors of one type, in which it is
    computed also under torch.autocast."""
    return _PackedMlpBlock.apply(x, a, weight, w_gate, w_up, w_down, eps)


# ---------------------------------------------------------------------------------------------
# The loss
# ---------------------------------------------------------------------------------------------
def fused_next_token_loss(logits: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """Mean cross entropy (fp32) of the token at t + 1 under logits[:, t]; labels of ``ignore_index`` do not count
    (NaN where none counts).  Under autograd the gradient is formed together with the loss, in one reading of the
    logits, and handed out by the first backward pass (a second one through the same loss is refused).  A loss that is
    scaled before its backward pass, such as ``loss / steps``, has that gradient read, multiplied and written once more, and
    rounded once more unless the factor is a power of two."""
    if torch.is_grad_enabled() and logits.requires_grad:
        return _lib.native().loss_autograd(logits, labels, ignore_index)
    return ops.next_token_loss(logits, labels, ignore_index, want_grad=False)[0]
