"""Linear attention over the state pool: what a GDN layer runs between its
projections (muserve/model/qwen35_layer_v2.py:163-201,286-295,351-358).

* ``causal_conv_prefill``: the causal conv of packed prompts, from and to the
  conv slots (``StatePool.conv_decode`` is its single-token form);
* ``linear_attn_prefill`` and ``linear_attn_decode``: linear attention with a
  decay for each head, by the delta rule or without it, over packed prompts and
  for single tokens, from and to the recurrent-state slots;
* ``gated_rms_norm``: the norm behind them (which both can apply themselves).

State tensors are one layer's slots: ``StatePool.state[layer]`` and
``StatePool.conv[layer]``; ``StatePool`` has the same calls by layer. A value
head's state is [128 values, 128 keys] fp32; value head h reads key head
h // (Hv / Hk). Sums, norms, gates and states are fp32, outputs are rounded to
bf16.

Calls are asynchronous on the current stream of the tensors' device. Data
faults (a slot outside the pool, offsets that do not hold together) set bits in
a per-device error word that ``check_errors(device)`` raises.
"""
from __future__ import annotations

import functools

import torch

from muserve_amd import _lib

HEAD_DIM = 128

_errors: dict[torch.device, _lib.DeviceErrors] = {}


def _errword(dev: torch.device) -> _lib.DeviceErrors:
    if dev not in _errors:
        _errors[dev] = _lib.DeviceErrors(dev)
    return _errors[dev]


def check_errors(device: torch.device | str = "cuda") -> None:
    """Raises MkvDeviceError for faults flagged by earlier calls (synchronises)."""
    dev = torch.device(device)
    if dev.type == "cuda" and dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    if dev in _errors:
        _errors[dev].check("linear attention")


def _call(dev: torch.device, name: str, *args) -> None:
    """The entry point on the current stream of ``dev``, also where another
    device is the current one."""
    if torch.cuda.current_device() == dev.index:
        _lib.call(name, *args, _lib.stream_of(dev))
    else:
        with torch.cuda.device(dev):
            _lib.call(name, *args, _lib.stream_of(dev))


# What a call's arguments come to, by their types, shapes, strides and devices
# alone: checking them anew takes 9 us, as long as a small call's kernel.
_plans: dict[tuple, tuple] = {}
_PLANS = 4096


def _sig(t: torch.Tensor | None):
    return None if t is None else (t.dtype, t.shape, t.stride(), t.get_device())


def _span(t: torch.Tensor | None) -> int:
    """Bytes from the first element of t to behind the last."""
    if t is None or t.numel() == 0:
        return 0
    return (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _apart(out: torch.Tensor, others, spans, names=("q", "k", "v", "g", "beta", "z")) -> None:
    """out is written while other workgroups still read."""
    at = out.data_ptr()
    end = at + out.numel() * out.element_size()
    for t, n, name in zip(others, spans, names):
        if n and t.data_ptr() < end and at < t.data_ptr() + n:
            raise ValueError(f"out must not be {name} or overlap it: other rows of it are still "
                             "to be read")


def _like(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape (torch.empty takes twice as long)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _planned(key: tuple, check, *args) -> tuple:
    plan = _plans.get(key)
    if plan is None:
        plan = check(*args)  # (raises for what is refused)
        if len(_plans) >= _PLANS:
            _plans.clear()
        _plans[key] = plan
    return plan


def _rows(name: str, t: torch.Tensor, heads: int, dim: int) -> int:
    """Bytes between the token rows of t [tokens, heads, dim] bf16, whose heads
    follow each other."""
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bf16, not {t.dtype}")
    if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim:
        raise ValueError(f"{name} must be [tokens, {heads}, {dim}], not {tuple(t.shape)}")
    if t.numel() == 0:
        return heads * dim * 2
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != dim):
        raise ValueError(f"{name}: the heads of a token must follow each other")
    if t.shape[0] == 1:
        return heads * dim * 2
    if t.stride(0) < heads * dim:
        raise ValueError(f"{name}: its rows overlap")
    return t.stride(0) * 2


def _gate(name: str, t: torch.Tensor, tokens: int, heads: int, dtype: torch.dtype) -> int:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, as g is, not {t.dtype}")
    if t.shape != (tokens, heads):
        raise ValueError(f"{name} must be [{tokens}, {heads}], not {tuple(t.shape)}")
    if t.numel() and heads > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the heads of a token must follow each other")
    if tokens <= 1:
        return heads * t.element_size()
    if t.stride(0) < heads:
        raise ValueError(f"{name}: its rows overlap")
    return t.stride(0) * t.element_size()


def _ids(name: str, t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    if t.dtype is torch.int32 and t.get_device() == dev.index and t.dim() == 1 \
            and t.is_contiguous():
        return t
    if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be a list of int32 (or int64) values")
    if t.dtype != torch.int32 or t.device != dev:
        t = t.to(device=dev, dtype=torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def _weight(w: torch.Tensor, dim: int) -> int:
    if w.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"the norm's weight must be bf16 or fp32, not {w.dtype}")
    if w.shape != (dim,) or not w.is_contiguous():
        raise ValueError(f"the norm's weight must be contiguous [{dim}]")
    return 1 if w.dtype == torch.bfloat16 else 0


def _check_common(q, k, v, g, beta, state, slots, a_log, dt_bias, z, norm_weight, out):
    """What both forms check: (device, tokens, key heads, value heads, pool
    slots, sizes of the inputs, their strides and types)."""
    dev = _lib.require_gpu(q, k, v, g, beta, state, a_log, dt_bias, z, norm_weight, out)
    if state.dtype != torch.float32 or state.dim() != 4 or not state.is_contiguous():
        raise ValueError("state must be contiguous fp32 [slots, value heads, 128, 128]")
    hv, hk = state.shape[1], k.shape[1] if k.dim() == 3 else 0
    if state.shape[2:] != (HEAD_DIM, HEAD_DIM):
        raise ValueError(f"unsupported state {tuple(state.shape)} (128 values x 128 keys)")
    if hk == 0 or hv % hk:
        raise ValueError(f"{hv} value heads do not share {hk} key heads evenly")
    if q.shape[0] != k.shape[0] or q.shape[0] != v.shape[0]:
        raise ValueError("q, k and v must have the same tokens")
    tokens = q.shape[0]
    qs, ks, vs = (_rows("q", q, hk, HEAD_DIM), _rows("k", k, hk, HEAD_DIM),
                  _rows("v", v, hv, HEAD_DIM))
    if g.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"g must be fp32 or bf16, not {g.dtype}")
    gs = _gate("g", g, tokens, hv, g.dtype)
    bs = 0 if beta is None else _gate("beta", beta, tokens, hv, g.dtype)
    if (a_log is None) != (dt_bias is None):
        raise ValueError("a_log and dt_bias come together")
    for name, t in (("a_log", a_log), ("dt_bias", dt_bias)):
        if t is not None and (t.dtype != torch.float32 or t.shape != (hv,)
                              or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous fp32 [{hv}]")
    if (z is None) != (norm_weight is None):
        raise ValueError("z and norm_weight come together")
    zs = wb = 0
    if z is not None:
        if z.shape[0] != tokens:
            raise ValueError("z must have the tokens of q")
        zs, wb = _rows("z", z, hv, HEAD_DIM), _weight(norm_weight, HEAD_DIM)
    if out is not None and (out.shape != (tokens, hv, HEAD_DIM) or out.dtype != torch.bfloat16
                            or not out.is_contiguous()):
        raise ValueError(f"out must be contiguous bf16 [{tokens}, {hv}, {HEAD_DIM}]")
    spans = tuple(_span(t) for t in (q, k, v, g, beta, z))
    return (dev, tokens, hk, hv, state.shape[0], spans, qs, ks, vs, gs, bs, zs, wb,
            1 if g.dtype == torch.bfloat16 else 0)


def _common(q, k, v, g, beta, state, slots, a_log, dt_bias, z, norm_weight, out):
    key = (_sig(q), _sig(k), _sig(v), _sig(g), _sig(beta), _sig(state), _sig(a_log), _sig(dt_bias),
           _sig(z), _sig(norm_weight), _sig(out))
    return _planned(key, _check_common, q, k, v, g, beta, state, slots, a_log, dt_bias, z,
                    norm_weight, out)


def _args(plan, q, k, v, g, beta, a_log, dt_bias, qk_norm, scale, z, norm_weight, eps, out):
    """The library's arguments from q on, up to out."""
    qs, ks, vs, gs, bs, zs, wb, gates_bf16 = plan[6:]
    return (q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, g.data_ptr(), gs,
            None if beta is None else beta.data_ptr(), bs, gates_bf16,
            None if a_log is None else a_log.data_ptr(),
            None if dt_bias is None else dt_bias.data_ptr(), 1 if qk_norm else 0,
            HEAD_DIM ** -0.5 if scale is None else float(scale),
            None if z is None else z.data_ptr(), zs,
            None if norm_weight is None else norm_weight.data_ptr(), wb, float(eps),
            out.data_ptr())


def linear_attn_decode(
    q: torch.Tensor,             # [B, Hk, 128] bf16
    k: torch.Tensor,             # [B, Hk, 128] bf16
    v: torch.Tensor,             # [B, Hv, 128] bf16
    g: torch.Tensor,             # [B, Hv] fp32 / bf16: log decay
    beta: torch.Tensor | None,   # [B, Hv] as g: write strength; None: no delta rule
    state: torch.Tensor,         # [slots, Hv, 128, 128] fp32, values x keys; updated in place
    slots: torch.Tensor,         # [B] int32, unique
    *,
    a_log: torch.Tensor | None = None,        # [Hv] fp32
    dt_bias: torch.Tensor | None = None,      # [Hv] fp32
    qk_norm: bool = False,
    scale: float | None = None,               # default 128 ** -0.5
    z: torch.Tensor | None = None,            # [B, Hv, 128] bf16
    norm_weight: torch.Tensor | None = None,  # [128] bf16 / fp32
    norm_eps: float = 1e-6,
    out: torch.Tensor | None = None,
    errors: _lib.DeviceErrors | None = None,
) -> torch.Tensor:               # [B, Hv, 128] bf16
    """One token per request (``gated_delta_rule_decode``,
    muserve/model/qwen35_layer_v2.py:286-295, on the slots themselves): with S
    the state of request b and head h,

        S <- exp(g) S;  u = beta (v - S k)  (u = v without beta)
        S <- S + u k^T;  out = scale S q

    ``qk_norm`` divides q and k by sqrt(|.|^2 + 1e-6) first. With ``a_log`` and
    ``dt_bias`` g and beta are the layer's projections:
    g = -exp(a_log) softplus(g + dt_bias), beta = sigmoid(beta). With ``z`` and
    ``norm_weight`` the output is o / sqrt(mean(o^2) + norm_eps) * norm_weight
    * silu(z). q, k, v and z may be views with strided token rows. A slot
    outside the pool gives zeros and a device fault; slots must be unique."""
    plan = _common(q, k, v, g, beta, state, slots, a_log, dt_bias, z, norm_weight, out)
    dev, B, hk, hv, pool = plan[:5]
    slots = _ids("slots", slots, dev)
    if out is None:
        out = _like(v)
    else:
        _apart(out, (q, k, v, g, beta, z), plan[5])
    if slots.numel() != B:
        raise ValueError(f"slots must name a slot for each of {B} requests")
    _call(dev, "mkv_linear_attn_decode", state.data_ptr(), pool, hk, hv, HEAD_DIM,
          slots.data_ptr(), B,
          *_args(plan, q, k, v, g, beta, a_log, dt_bias, qk_norm, scale, z, norm_weight, norm_eps,
                 out), (errors or _errword(dev)).ptr())
    return out


@functools.lru_cache(maxsize=1024)
def _prefill_bytes(tokens: int, batch: int, max_seqlen: int, hk: int, hv: int, delta: bool,
                   dev: torch.device) -> int:
    n = _lib.load().mkv_linear_attn_prefill_workspace_bytes(tokens, batch, max_seqlen, hk, hv,
                                                            1 if delta else 0)
    if n < 0:
        raise ValueError("bad linear attention shape")
    return n


def linear_attn_prefill(
    q: torch.Tensor,             # [total_tokens, Hk, 128] bf16
    k: torch.Tensor,             # [total_tokens, Hk, 128] bf16
    v: torch.Tensor,             # [total_tokens, Hv, 128] bf16
    g: torch.Tensor,             # [total_tokens, Hv] fp32 / bf16
    beta: torch.Tensor | None,   # [total_tokens, Hv] as g, or None
    state: torch.Tensor,         # [slots, Hv, 128, 128] fp32; updated in place
    slots: torch.Tensor,         # [num_seqs] int32, unique
    cu_seqlens: torch.Tensor,    # [num_seqs + 1] int32
    *,
    max_seqlen: int | None = None,
    a_log: torch.Tensor | None = None,
    dt_bias: torch.Tensor | None = None,
    qk_norm: bool = False,
    scale: float | None = None,
    z: torch.Tensor | None = None,
    norm_weight: torch.Tensor | None = None,
    norm_eps: float = 1e-6,
    out: torch.Tensor | None = None,
    errors: _lib.DeviceErrors | None = None,
) -> torch.Tensor:               # [total_tokens, Hv, 128] bf16
    """``linear_attn_decode``'s recurrence over packed prompts
    (``chunk_gated_delta_rule``, muserve/model/qwen35_layer_v2.py:351-358):
    sequence b is rows cu_seqlens[b]..cu_seqlens[b+1], starts from the state in
    slots[b] (``StatePool.reset`` for a new request; a later chunk of a prompt
    goes on where the last one ended) and leaves its final state there. Rows of
    ``out`` outside the sequences are left as they were. ``max_seqlen`` (the
    longest sequence, if the caller knows it) helps to choose the form of the
    computation. Offsets that do not hold together are a device fault, and the
    call then writes nothing."""
    plan = _common(q, k, v, g, beta, state, slots, a_log, dt_bias, z, norm_weight, out)
    dev, tokens, hk, hv, pool = plan[:5]
    slots = _ids("slots", slots, dev)
    if out is None:
        out = _like(v)
    else:
        _apart(out, (q, k, v, g, beta, z), plan[5])
    cu = _ids("cu_seqlens", cu_seqlens, dev)
    batch = slots.numel()
    if cu.numel() != batch + 1:
        raise ValueError(f"cu_seqlens must hold {batch + 1} offsets for {batch} slots")
    longest = 0 if max_seqlen is None else int(max_seqlen)
    if longest < 0:
        raise ValueError("max_seqlen must not be negative")
    longest = min(longest or tokens, tokens)
    # from torch's allocator at each call, which orders its reuse by stream and
    # keeps it with a graph under capture
    need = _prefill_bytes(tokens, batch, longest, hk, hv, beta is not None, dev)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(dev, "mkv_linear_attn_prefill", state.data_ptr(), pool, hk, hv, HEAD_DIM,
          slots.data_ptr(), cu.data_ptr(), batch, tokens, longest,
          *_args(plan, q, k, v, g, beta, a_log, dt_bias, qk_norm, scale, z, norm_weight, norm_eps,
                 out), ws.data_ptr(), need, (errors or _errword(dev)).ptr())
    return out


def _check_conv(x, weight, conv_state, out):
    dev = _lib.require_gpu(x, weight, conv_state, out)
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16 \
            or conv_state.dtype != torch.bfloat16:
        raise TypeError("causal_conv_prefill takes bf16 x, weight and conv states")
    if conv_state.dim() != 3 or not conv_state.is_contiguous():
        raise ValueError("conv_state must be contiguous [slots, channels, width]")
    C, W = conv_state.shape[1], conv_state.shape[2]
    if x.dim() != 2 or x.shape[1] != C:
        raise ValueError(f"x must be [tokens, {C}], not {tuple(x.shape)}")
    T = x.shape[0]
    if x.numel() and (x.stride(1) != 1 or (T > 1 and x.stride(0) < C)):
        raise ValueError("x: the channels of a token must follow each other")
    if weight.dim() not in (2, 3) or weight.shape[0] != C or weight.numel() != C * weight.shape[-1]:
        raise ValueError(f"weight must be [{C}, 1, K] or [{C}, K]")
    if out is not None and (out.shape != (T, C) or out.dtype != x.dtype
                            or not out.is_contiguous()):
        raise ValueError(f"out must be contiguous bf16 [{T}, {C}]")
    return dev, T, C, W, weight.shape[-1], x.stride(0) * 2 if T > 1 else C * 2, (_span(x),)


def causal_conv_prefill(
    x: torch.Tensor,           # [total_tokens, C] bf16
    weight: torch.Tensor,      # [C, 1, 4] or [C, 4] bf16
    conv_state: torch.Tensor,  # [slots, C, 3 or 4] bf16; updated in place
    slots: torch.Tensor,       # [num_seqs] int32, unique
    cu_seqlens: torch.Tensor,  # [num_seqs + 1] int32
    *,
    out: torch.Tensor | None = None,
    errors: _lib.DeviceErrors | None = None,
) -> torch.Tensor:             # [total_tokens, C] bf16
    """The causal conv of packed prompts (muserve/model/qwen35_layer_v2.py:
    163-201, prefill branch): out[t] = silu(sum_k weight[:, k] x[t - 3 + k])
    for each channel, the inputs before a sequence's first row taken from
    slots[b], which is left with the sequence's last inputs. Rows of x may be
    strided; rows of ``out`` outside the sequences are left as they were."""
    key = (_sig(x), _sig(weight), _sig(conv_state), _sig(out))
    dev, T, C, W, K, xs, spans = _planned(key, _check_conv, x, weight, conv_state, out)
    w = weight if weight.is_contiguous() else weight.contiguous()
    if out is None:
        out = _like(x)
    else:
        _apart(out, (x,), spans, ("x",))
    slots, cu = _ids("slots", slots, dev), _ids("cu_seqlens", cu_seqlens, dev)
    batch = slots.numel()
    if cu.numel() != batch + 1:
        raise ValueError(f"cu_seqlens must hold {batch + 1} offsets for {batch} slots")
    _call(dev, "mkv_gdn_conv_prefill", conv_state.data_ptr(), conv_state.shape[0], C, W,
          slots.data_ptr(), cu.data_ptr(), batch, T, x.data_ptr(), xs, w.data_ptr(), K,
          out.data_ptr(),
          (errors or _errword(dev)).ptr())
    return out


def _check_norm(x, z, weight, out):
    dev = _lib.require_gpu(x, z, weight, out)
    if x.dim() not in (2, 3) or z.shape != x.shape:
        raise ValueError(f"x and z must be [tokens, heads, D] or [rows, D] alike, not "
                         f"{tuple(x.shape)} and {tuple(z.shape)}")
    D = x.shape[-1]
    if D == 0 or D % 8 or D > 4096:
        raise ValueError(f"unsupported rows of {D} values (a multiple of 8, at most 4096)")
    x3, z3 = (x, z) if x.dim() == 3 else (x.unsqueeze(1), z.unsqueeze(1))
    T, H = x3.shape[:2]
    xs, zs, wb = _rows("x", x3, H, D), _rows("z", z3, H, D), _weight(weight, D)
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype
                            or not out.is_contiguous()):
        raise ValueError("out must be a contiguous tensor shaped like x")
    # (out may lie on x or z without gaps: a thread reads what it writes)
    whole = H * D * 2
    return (dev, T if H else 0, H, D, xs, zs, wb, (_span(x), _span(z)),
            (xs == whole, zs == whole))


def gated_rms_norm(
    x: torch.Tensor,       # [tokens, heads, D] or [rows, D] bf16
    z: torch.Tensor,       # as x
    weight: torch.Tensor,  # [D] bf16 / fp32
    eps: float = 1e-6,
    *,
    out: torch.Tensor | None = None,
) -> torch.Tensor:         # as x
    """x / sqrt(mean(x^2) + eps) * weight * silu(z) over the last dimension (a
    multiple of 8, at most 4096), in fp32, rounded once. The rows of a token
    follow each other; tokens may be strided. ``out`` may be x or z."""
    key = (_sig(x), _sig(z), _sig(weight), _sig(out))
    dev, T, H, D, xs, zs, wb, spans, whole = _planned(key, _check_norm, x, z, weight, out)
    if out is None:
        out = _like(x)
    else:
        at = out.data_ptr()
        _apart(out, (x, z), [0 if w and t.data_ptr() == at else n
                             for t, w, n in zip((x, z), whole, spans)], ("x", "z"))
    if T:
        _call(dev, "mkv_gated_rms_norm", x.data_ptr(), xs, z.data_ptr(), zs, T, H, D,
              weight.data_ptr(), wb, float(eps), out.data_ptr())
    return out
