"""The norm of each query and key head and the rotation by its position
(muserve/model/qwen35_layer_v2.py:458-469), in one pass.

* ``qk_norm_rope``: q and k of any strides to new (or given) tensors;
* ``PagedKVCache.append_rope``: the same with K and V written straight into the
  pool's pages, of any of its types.

Norms, angles (in fp64) and products are fp32; each output is rounded once.
Calls are asynchronous on the current stream of the tensors' device.
"""
from __future__ import annotations

import torch

from muserve_amd import _lib

HEAD_DIMS = (64, 128, 256)
_WEIGHT_KINDS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}

# What a call's arguments come to, by their types, shapes, strides and devices
# alone (checking them anew takes longer than a small call's kernel).
_plans: dict[tuple, tuple] = {}
_PLANS = 4096


def _heads(name: str, t: torch.Tensor, tokens: int, dim: int, dtype: torch.dtype):
    """(heads, bytes between tokens, bytes between heads) of t [tokens, heads, dim]."""
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != dim:
        raise ValueError(f"{name} must be [{tokens}, heads, {dim}], not {tuple(t.shape)}")
    heads = t.shape[1]
    if t.numel() == 0:
        return heads, 0, 0
    if t.stride(2) != 1 or (tokens > 1 and t.stride(0) % 8) or (heads > 1 and t.stride(1) % 8):
        raise ValueError(f"{name}: the dims of a head must follow each other, its rows start at "
                         "multiples of 8 elements")
    return (heads, 2 * t.stride(0) if tokens > 1 else 0, 2 * t.stride(1) if heads > 1 else 0)


def _check(q, k, v, positions, inv_freq, q_weight, k_weight, interleaved):
    """The call's constants: (device, tokens, arguments ahead of the weights)."""
    dev = _lib.require_gpu(q, k, v, positions, inv_freq, q_weight, k_weight)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"q and k must be bf16 or fp16, not {q.dtype}")
    if q.dim() != 3 or q.shape[2] not in HEAD_DIMS:
        raise ValueError(f"q must be [tokens, heads, 64, 128 or 256], not {tuple(q.shape)}")
    tokens, hq, dim = q.shape
    _, q_token, q_head = _heads("q", q, tokens, dim, q.dtype)
    hk, k_token, k_head = _heads("k", k, tokens, dim, q.dtype)
    strides = (0, 0)
    if v is not None:
        if v.shape != k.shape:
            raise ValueError(f"v must be {tuple(k.shape)} as k is, not {tuple(v.shape)}")
        strides = _heads("v", v, tokens, dim, q.dtype)[1:]
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (tokens,):
        raise ValueError(f"positions must be int32 or int64 [{tokens}]")
    if inv_freq.dtype not in (torch.float32, torch.float64) or inv_freq.dim() != 1 \
            or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous fp32 or fp64 [rotary_dim / 2]")
    rot = 2 * inv_freq.numel()
    if rot == 0 or rot % 16 or rot > dim:
        raise ValueError(f"rotary dim {rot} unsupported (multiples of 16 up to {dim})")
    kind = 0
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if w.dtype not in _WEIGHT_KINDS or w.shape != (dim,) or not w.is_contiguous():
            raise ValueError(f"{name} must be contiguous bf16, fp16 or fp32 [{dim}]")
        if kind and kind != _WEIGHT_KINDS[w.dtype]:
            raise TypeError("q_weight and k_weight must be of one type")
        kind = _WEIGHT_KINDS[w.dtype]
    name, at = ("mkv_qk_norm_rope", 6) if v is None else ("mkv_append_rope", 9)
    direct = positions.dtype == torch.int64 and positions.is_contiguous()
    return (dev, direct, _lib.constants(name, 1, q_token, q_head),
            _lib.constants(name, 4, k_token, k_head), _lib.constants(name, 7, *strides),
            _lib.constants(name, at, tokens, hq, hk, dim, 1 if q.dtype == torch.float16 else 0),
            _lib.constants(name, at + 7, 1 if inv_freq.dtype == torch.float64 else 0, rot,
                           1 if interleaved else 0), kind)


def _plan(q, k, v, positions, inv_freq, q_weight, k_weight, interleaved):
    # (attributes in a row: a helper for each tensor costs half as much again)
    key = (q.dtype, q.shape, q.stride(), q.get_device(), k.dtype, k.shape, k.stride(),
           k.get_device(), positions.dtype, positions.shape, positions.is_contiguous(),
           positions.get_device(), inv_freq.dtype, inv_freq.shape, inv_freq.is_contiguous(),
           inv_freq.get_device(), interleaved,
           None if q_weight is None else (q_weight.dtype, q_weight.shape,
                                          q_weight.is_contiguous(), q_weight.get_device()),
           None if k_weight is None else (k_weight.dtype, k_weight.shape,
                                          k_weight.is_contiguous(), k_weight.get_device()),
           None if v is None else (v.dtype, v.shape, v.stride(), v.get_device()))
    plan = _plans.get(key)
    if plan is None:
        plan = _check(q, k, v, positions, inv_freq, q_weight, k_weight, interleaved)
        if len(_plans) >= _PLANS:
            _plans.clear()
        _plans[key] = plan
    return plan


def _given(name: str, out: torch.Tensor, own: torch.Tensor, others) -> None:
    """An output that the caller gives: contiguous, and its own input itself or apart from
    everything that other rows still read."""
    if out.shape != own.shape or out.dtype != own.dtype or out.device != own.device \
            or not out.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of its input's shape and type")
    if out.data_ptr() != own.data_ptr() or not own.is_contiguous():
        others = (own, *others)  # (also where another input is the same tensor as its own)
    lo, hi = _lib.span(out)
    for t in others:
        if t is None:
            continue
        a, b = _lib.span(t)
        if a < hi and lo < b:
            raise ValueError(f"{name} overlaps a tensor that other rows still read or write")


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def qk_norm_rope(
    q: torch.Tensor,                      # [tokens, NUM_Q_HEADS, head_dim] bf16 / fp16
    k: torch.Tensor,                      # [tokens, NUM_KV_HEADS, head_dim] same
    positions: torch.Tensor,              # [tokens] int64 (plan.positions) or int32
    inv_freq: torch.Tensor,               # [rotary_dim / 2] fp32 or fp64
    q_weight: torch.Tensor | None = None,  # [head_dim] bf16, fp16 or fp32
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    *,
    rope_scale: float = 1.0,
    zero_centered: bool = False,
    interleaved: bool = False,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head of q and k with their weights (one is added to
    them with ``zero_centered``; no norm where a weight is None), then the
    rotation of the first ``rotary_dim`` dims by ``positions * inv_freq``: dim i
    with dim ``i + rotary_dim / 2``, or dims 2i and 2i + 1 (``interleaved``);
    ``rope_scale`` multiplies sines and cosines.

    head_dim 64, 128 or 256, rotary_dim a multiple of 16. q and k may be views
    of a projection's output (dims contiguous, rows at multiples of 8
    elements); the outputs are contiguous, and ``out`` may be the inputs
    themselves where those are."""
    plan = _plan(q, k, None, positions, inv_freq, q_weight, k_weight, interleaved)
    dev, direct, q_strides, k_strides, _, sizes, freq, kind = plan
    if out is None:
        q_out, k_out = _like(q), _like(k)
    else:
        q_out, k_out = out
        _given("out[0]", q_out, q, (k, positions, inv_freq, q_weight, k_weight))
        _given("out[1]", k_out, k, (q, q_out, positions, inv_freq, q_weight, k_weight))
    if not direct:
        positions = positions.long().contiguous()
    _lib.call_on(dev, "mkv_qk_norm_rope", q.data_ptr(), *q_strides, k.data_ptr(), *k_strides,
                 *sizes, positions.data_ptr(), inv_freq.data_ptr(), *freq, rope_scale,
                 None if q_weight is None else q_weight.data_ptr(),
                 None if k_weight is None else k_weight.data_ptr(), kind, 1 if zero_centered else 0,
                 eps, q_out.data_ptr(), k_out.data_ptr())
    return q_out, k_out


POOL_16, POOL_FP8, POOL_FP4 = 1, 2, 3


def append_rope(q, k, v, positions, inv_freq, q_weight, k_weight, eps, rope_scale, zero_centered,
                interleaved, out, slots, pool, errors, cache, scales):
    """``PagedKVCache.append_rope`` once the pool is known: ``pool`` is (type,
    K plane, V plane, K scales, V scales, slots) by address, of the tensors
    ``cache`` and ``scales``."""
    plan = _plan(q, k, v, positions, inv_freq, q_weight, k_weight, interleaved)
    dev, direct, q_strides, k_strides, v_strides, sizes, freq, kind = plan
    if out is None:
        out = _like(q)
    else:
        _given("out", out, q, (k, v, positions, inv_freq, q_weight, k_weight, slots, cache, scales))
    if not direct:
        positions = positions.long().contiguous()
    _lib.call_on(dev, "mkv_append_rope", q.data_ptr(), *q_strides, k.data_ptr(), *k_strides,
                 v.data_ptr(), *v_strides, *sizes, positions.data_ptr(), inv_freq.data_ptr(), *freq,
                 rope_scale, None if q_weight is None else q_weight.data_ptr(),
                 None if k_weight is None else k_weight.data_ptr(), kind,
                 1 if zero_centered else 0, eps, out.data_ptr(), *pool, slots.data_ptr(),
                 errors.word.data_ptr())
    return out
