"""Inputs and error bounds of the linear-attention tests."""
import torch

from oracle import linear as ref
from tests.gpu_util import DEV

D = 128
HALF_BF16 = 2.0 ** -8  # half a rounding step, relative
U32 = 2.0 ** -24


def inputs(seed, tokens, hk, hv, *, raw=True, delta=True, qk_norm=True, norm=False, slots=1,
           strided=True, wide=False):
    """CPU tensors of a call. q, k and v are views of one row buffer."""
    gen = torch.Generator().manual_seed(seed)

    def normal(*size):
        return torch.randn(*size, generator=gen)

    pad = 64 if wide else 0
    mixed = torch.nn.functional.silu(normal(tokens, (2 * hk + hv) * D + pad))
    if not qk_norm:
        qk = mixed[:, :2 * hk * D].view(tokens, 2 * hk, D)
        qk /= (qk.square().sum(-1, keepdim=True) + 1e-6).sqrt()
    mixed = mixed.bfloat16()
    x = {"mixed": mixed, "hk": hk, "hv": hv, "qk_norm": qk_norm}
    if raw:
        x["g"] = normal(tokens, hv).bfloat16()
        x["beta"] = normal(tokens, hv).bfloat16()
        x["a_log"] = (1 + 15 * torch.rand(hv, generator=gen)).log()
        x["dt_bias"] = normal(hv) - 3
    else:
        x["g"] = -(0.001 + 0.5 * torch.rand(tokens, hv, generator=gen) ** 2)
        x["beta"] = torch.rand(tokens, hv, generator=gen)
        x["a_log"] = x["dt_bias"] = None
    if not delta:
        x["beta"] = None
    x["z"] = normal(tokens, hv, D).bfloat16() if norm else None
    x["w"] = (1 + 0.2 * normal(D)).bfloat16() if norm else None
    x["state"] = 0.2 * normal(slots, hv, D, D)
    return x


def split(mixed, hk, hv):
    t = mixed.shape[0]
    return (mixed[:, :hk * D].view(t, hk, D), mixed[:, hk * D:2 * hk * D].view(t, hk, D),
            mixed[:, 2 * hk * D:(2 * hk + hv) * D].view(t, hv, D))


def on_gpu(x):
    return {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in x.items()}


def keywords(x, eps=1e-6):
    return {"a_log": x["a_log"], "dt_bias": x["dt_bias"], "qk_norm": x["qk_norm"], "z": x["z"],
            "norm_weight": x["w"], "norm_eps": eps}


def want_sequence(x, rows, state, scale=D ** -0.5):
    """The oracle on rows `rows` (a slice) from `state` [Hv, D, D]: outputs,
    final state, and the bounds of both.

    Rounding errors of a state: every token multiplies S by (I - beta k k^T) e^g,
    which does not grow its norm (0 <= beta <= 1, |k| <= 1, g <= 0), and adds an
    error of its own: sums of at most 128 + 64 products and a few roundings of
    terms no larger than |S| + |u|. Independent roundings of 2^-24 add up as the
    root of their number: sqrt(192) a token, sqrt(T) tokens; 8 of these leave
    nothing to chance. An output adds scale |q| times that, its own sum of 192
    products, and its rounding to bf16."""
    q, k, v = (t[rows] for t in split(x["mixed"], x["hk"], x["hv"]))
    beta = None if x["beta"] is None else x["beta"][rows]
    o, s, size = ref.scan(q, k, v, x["g"][rows], beta, state, scale, x["qk_norm"], x["a_log"],
                          x["dt_bias"])
    steps = max(1, v.shape[0])
    s_tol = 8 * U32 * (192 * steps) ** 0.5 * size
    qn = ref.normed(q, x["qk_norm"]).norm(dim=-1).repeat_interleave(x["hv"] // x["hk"], 1)
    o_tol = abs(scale) * qn * s_tol * 2
    o_tol = o_tol[:, :, None].expand_as(o)
    return o, s, s_tol, o_tol


def with_norm(x, rows, o, o_tol, eps=1e-6, rounded=False):
    """The gated norm of the oracle's outputs and its bound: an error d of o
    moves y by d / rms |w silu(z)|, and the rms by at most the rms of d."""
    if rounded:
        o_tol = o_tol + HALF_BF16 * o.abs()
    z, w = x["z"][rows], x["w"]
    y = ref.gated_norm(o, z, w, eps)
    zz = z.double()
    rms = (o.square().mean(-1, keepdim=True) + eps).sqrt()
    gain = (w.double() * zz * torch.sigmoid(zz)).abs() / rms
    d = (o_tol.square().mean(-1, keepdim=True)).sqrt()
    return y, gain * o_tol + y.abs() * (d / rms + 32 * U32)


def close(got, want, tol, what):
    """bf16 outputs: `tol` and half a rounding step of a value within it."""
    err = (got.double().cpu() - want).abs()
    bound = tol + HALF_BF16 * (want.abs() + tol) + 2.0 ** -133
    assert torch.isfinite(got.float()).all(), f"{what}: not finite"
    worst = (err / bound).max() if err.numel() else 0
    assert (err <= bound).all(), f"{what}: {float(worst):.3g} times the bound"


def close_state(got, want, tol, what):
    """fp32 states by head, in the norm of the bound."""
    err = (got.double().cpu() - want).flatten(-2).norm(dim=-1)
    assert (err <= tol).all(), f"{what}: {float((err / tol).max()):.3g} times the bound"
