"""3D RoPE tables and dynamic time remaps.

* ``rope_params`` / ``wan_freqs``: the Wan table definition
  (wan/modules/model.py:29-36; t/h/w concat causal_model.py:585-590):
  row p, pair j = exp(i * p * theta^(-2j/dim)) in float64.
* ``split_freqs`` / ``flat_freq_parts``: the 22/21/21 split and the fp32
  (re, im) interleaved tables the pack kernel reads
  (pyramidkv/_mega_cache.py:713-731).
* ``apply_rope_to_flat_k``: rotates packed K on the GPU
  (torch.ops.adahead.rope_apply); replaces rope.py:18-68 and the Triton
  kernel of triton_rope.py.
* ``map_sink_time`` / ``map_dynamic_pos_time``: rope.py:86-134.
* ``rotary`` / ``rotary_frequencies``: rotation of q and k heads at any
  position, without a table: both pair layouts, part of a head, one or several
  position axes, frequencies scaled for long contexts, with its gradient.
"""
from __future__ import annotations

import math

import torch
from torch.autograd import forward_ad

from . import _ops


def rope_params(max_seq_len: int, dim: int, theta: float = 10000) -> torch.Tensor:
    assert dim % 2 == 0
    ang = torch.outer(torch.arange(max_seq_len, dtype=torch.float64),
                      1.0 / torch.pow(theta, torch.arange(0, dim, 2, dtype=torch.float64).div(dim)))
    return torch.polar(torch.ones_like(ang), ang)


def wan_freqs(head_dim: int = 128, max_seq_len: int = 1024, theta: float = 10000) -> torch.Tensor:
    d = head_dim
    return torch.cat([rope_params(max_seq_len, d - 4 * (d // 6), theta),
                      rope_params(max_seq_len, 2 * (d // 6), theta),
                      rope_params(max_seq_len, 2 * (d // 6), theta)], dim=1)


def split_freqs(freqs: torch.Tensor):
    c = freqs.shape[1]
    return tuple(p.contiguous() for p in freqs.split([c - 2 * (c // 3), c // 3, c // 3], dim=1))


def flat_freq_parts(freqs: torch.Tensor, device=None):
    """(ft, fy, fx) fp32 [rows, cols*2] with (re, im) interleaved."""
    out = []
    for z in split_freqs(freqs):
        z = z.to(device=device) if device is not None else z
        out.append(torch.view_as_real(z.to(torch.complex64)).contiguous().view(z.shape[0], -1))
    return tuple(out)


def apply_rope_to_flat_k(k_flat: torch.Tensor, pos_3d: torch.Tensor, freqs: torch.Tensor,
                         freq_parts=None, out: torch.Tensor | None = None, freq_parts_flat=None) -> torch.Tensor:
    """Rotate k_flat [n, D] (bf16, on the GPU) at positions pos_3d [n, 3]."""
    if k_flat.numel() == 0:
        return out if out is not None else k_flat
    if k_flat.shape[1] % 2 != 0:
        raise ValueError(f"Head dim must be even, got {k_flat.shape[1]}")
    if freq_parts_flat is None:
        if freq_parts is not None:
            freq_parts_flat = tuple(torch.view_as_real(p.to(torch.complex64)).contiguous().view(p.shape[0], -1)
                                    .to(k_flat.device) for p in freq_parts)
        else:
            freq_parts_flat = flat_freq_parts(freqs, k_flat.device)
    res = _ops.ops().rope_apply(k_flat.contiguous(), pos_3d.to(device=k_flat.device, dtype=torch.long),
                                *freq_parts_flat)
    if out is not None:
        out.copy_(res)
        return out
    return res


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                       trained_length: int = 0, fast_turns: float = 32.0, slow_turns: float = 1.0, device=None):
    """(frequencies [rotary_dim / 2] float64, scale) for ``rotary``: pair j
    turns by theta^(-2j / rotary_dim) radians a position.  scaling, for contexts
    ``factor`` times as long as those trained on:

    * "linear": every frequency divided by the factor;
    * "base": theta raised so that the slowest pair is slowed by the factor and
      the fastest not at all;
    * "parts": pairs of more than ``fast_turns`` turns within ``trained_length``
      positions as they are, those of fewer than ``slow_turns`` divided by the
      factor, a linear blend by turns between them, and rotated q and k scaled
      by 0.1 ln(factor) + 1 each."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_frequencies: rotary_dim ({rotary_dim}) must be even and at least 2")
    if factor < 1.0:
        raise ValueError(f"rotary_frequencies: factor ({factor}) must be at least 1")
    j = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim
    if scaling == "base":
        if rotary_dim > 2:
            theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
        return theta ** -j, 1.0
    f = theta ** -j
    if scaling is None:
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling != "parts":
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}")
    if trained_length <= 0 or fast_turns <= slow_turns:
        raise ValueError("rotary_frequencies: parts needs trained_length, and fast_turns above slow_turns")
    turns = trained_length * f / (2 * math.pi)
    keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
    return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1.0


_transforms_active = torch._C._are_functorch_transforms_active


def _rotary_op(q, k, *args):
    out = _ops.ops().rotary(q, k, *args)
    return out[0] if k is None else tuple(out)


class _Rotary(torch.autograd.Function):
    """The rotation is linear: backwards it is the inverse rotation of the
    outputs' gradients, forwards the same one of the inputs' tangents."""

    @staticmethod
    def forward(ctx, *inputs):
        _Rotary.save(ctx, *inputs)
        return _rotary_op(*inputs)

    @staticmethod
    def save(ctx, q, k, positions, freqs, *args):
        ctx.save_for_backward(positions, freqs)
        ctx.save_for_forward(positions, freqs)
        ctx.args, ctx.q_shape, ctx.k_shape = args, q.shape, None if k is None else k.shape
        ctx.set_materialize_grads(False)

    @staticmethod
    def backward(ctx, gq, gk=None):
        axes, interleaved, scale, inverse = ctx.args
        return (*_turn(gq, gk, *ctx.saved_tensors, axes, interleaved, scale, not inverse), *(None,) * 6)

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        tq, tk = _turn(tq, tk, *ctx.saved_tensors, *ctx.args)
        if ctx.k_shape is None:
            return tq
        # (of two outputs both have a tangent)
        return tk.new_zeros(ctx.q_shape) if tq is None else tq, tq.new_zeros(ctx.k_shape) if tk is None else tk


class _RotaryTransformed(_Rotary):
    """Under torch.func, which asks for this form (43 us of host time a call, 14 in
    the other)."""

    @staticmethod
    def forward(q, k, positions, freqs, axes, interleaved, scale, inverse):
        return _rotary_op(q, k, positions, freqs, axes, interleaved, scale, inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _Rotary.save(ctx, *inputs)

    @staticmethod
    def vmap(info, in_dims, q, k, positions, freqs, *args):
        """The batch as more rows."""
        if in_dims[3] is not None:
            raise RuntimeError("rotary: freqs cannot be batched")
        n = info.batch_size

        def rows(x, dim):
            return (x.expand(n, *x.shape) if dim is None else x.movedim(dim, 0)).flatten(0, 1).contiguous()

        back = lambda x: x.view(n, x.shape[0] // n, *x.shape[1:])
        out = _rotary(rows(q, in_dims[0]), None if k is None else rows(k, in_dims[1]), rows(positions, in_dims[2]), freqs,
                      *args)
        return (back(out), 0) if k is None else (tuple(back(x) for x in out), (0, 0))


def _rotary(*args):
    return (_RotaryTransformed if _transforms_active() else _Rotary).apply(*args)


def _turn(q, k, *args):
    """q and k, either of which may be None, rotated."""
    dense = lambda x: x if x is None or x.stride(-1) == 1 else x.contiguous()
    q, k = dense(q), dense(k)
    if q is not None and k is not None:
        return _rotary(q, k, *args)
    if q is None and k is None:
        return None, None
    x = _rotary(k if q is None else q, None, *args)
    return (None, x) if q is None else (x, None)


def rotary(q: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, *, k: torch.Tensor | None = None, axes=None,
           interleaved: bool = True, scale: float = 1.0, inverse: bool = False):
    """Rotate the heads of q [rows, heads, D] (and of k, in the same launch) by
    their rows' positions; bf16, fp16 or fp32, slices of a fused projection as
    they lie.  Returns the rotated q, or (q, k).

    positions [rows] or [rows, A] (int64 or int32): the first axes[0] pairs of a
    head turn by the first column, the next axes[1] by the second, ... (default:
    all by one).  freqs: float64, one a pair (rotary_frequencies); angles are
    taken in 64 bits, so positions may be far.  Pair j is columns 2j and 2j + 1
    (interleaved) or j and j + pairs; columns from twice the pairs on are
    copied.  inverse turns back.  Differentiable in q and k, backwards, forwards
    (dual tensors) and under torch.func, vmap among it; not in freqs, which must
    not ask for a gradient.  A graph that captures the backward pass too needs
    leaves that no living eager result was computed from (torch ends the process
    otherwise)."""
    grad = torch.is_grad_enabled()
    if grad and freqs.requires_grad:
        raise RuntimeError("rotary: freqs have no gradient; detach them")
    axes = (int(freqs.numel()),) if axes is None else tuple(int(a) for a in axes)
    args = (positions, freqs, axes, bool(interleaved), float(scale), bool(inverse))
    # wherever a derivative may be asked for: gradients, dual tensors, torch.func
    if (grad and (q.requires_grad or (k is not None and k.requires_grad))) or forward_ad._current_level >= 0 or \
            _transforms_active():
        return _rotary(q, k, *args)
    return _rotary_op(q, k, *args)


def map_sink_time(sync_t_raw: int, sink_time_mapping_mode: str, sink_time_clamp_min: int,
                  sink_time_clamp_max: int, decoupled_sink_time_lag: int) -> int:
    if sink_time_mapping_mode == "window_clamp":
        delta = min(max(sync_t_raw, sink_time_clamp_min), sink_time_clamp_max)
        return max(0, sync_t_raw - delta)
    return max(0, sync_t_raw - decoupled_sink_time_lag)


def map_dynamic_pos_time(dyn_pos: torch.Tensor, current_t: int, history_time_mapping_mode: str,
                         history_relative_t_max: int, history_time_soft_factor: float,
                         inplace: bool = False) -> torch.Tensor:
    mode = history_time_mapping_mode
    if mode == "none" or history_relative_t_max <= 0:
        return dyn_pos
    if mode == "relative_softcap":
        mapped = dyn_pos if inplace else dyn_pos.clone()
        rel = (current_t - mapped[:, 0].long()).clamp(min=0)
        over = (rel - history_relative_t_max).clamp(min=0)
        comp = torch.round(over.to(torch.float32) * history_time_soft_factor).to(torch.long)
        rel_mapped = torch.where(rel <= history_relative_t_max, rel, history_relative_t_max + comp)
        mapped[:, 0] = (current_t - rel_mapped).clamp(min=0)
        return mapped
    if mode != "relative_clamp":
        return dyn_pos
    mapped = dyn_pos if inplace else dyn_pos.clone()
    rel = (current_t - mapped[:, 0].long()).clamp(min=0, max=history_relative_t_max)
    mapped[:, 0] = current_t - rel
    return mapped
