"""Timed cases of a linear-attention (GDN) layer's operators on one GPU, between
its projections: what a serving step runs for the layers whose states live in
slots of a state pool.

* ``step``: the recurrent form: one token per request, its state read from and
  written back to the request's slot, by the decay alone or by the delta rule,
  with the q / k norms, the gates and the output's gated norm as asked;
* ``prompt``: the chunked form over packed prompts, from and to their slots;
* ``conv``: the causal conv of packed prompts from and to the conv slots;
* ``norm``: the gated RMS norm after the layer.

With ``own`` unset ``run`` computes the operators with elementary torch
operations in fp32 (running sums of log decays in fp64), rounded once at the
end; with ``own`` set it calls the package. Sequence lengths and slots come
from the case; the seed makes the values.
"""
import math

import numpy as np
import torch

own = False

D = 128          # key and value dims of a head
CHUNK = 64       # tokens per chunk of the plain prompt form
MOST = 8 * 32768  # tokens x value heads of the largest prompt case
L2_EPS = 1e-6
EPS = 1e-6


def listed():
    return [
        # one interactive user's decode step on one rank of eight: latency and launches
        {"name": "step one user", "kind": "step", "batch": 1, "hk": 2, "hv": 8, "delta": True,
         "raw": True, "qk_norm": True, "norm": True, "shape": 1},
        # the serving loop's full decode batch on one rank
        {"name": "step full batch", "kind": "step", "batch": 256, "hk": 2, "hv": 8, "delta": True,
         "raw": True, "qk_norm": True, "norm": True, "shape": 2},
        # a decay alone, given by the caller, one key head per value head
        {"name": "step decay only", "kind": "step", "batch": 37, "hk": 8, "hv": 8, "delta": False,
         "raw": False, "qk_norm": False, "norm": False, "shape": 3},
        # a short chat turn: the smallest prompt
        {"name": "prompt short", "kind": "prompt", "seqs": 1, "median": 77, "sigma": 0.0, "hk": 2,
         "hv": 8, "delta": True, "raw": True, "qk_norm": True, "norm": False, "shape": 4},
        # a mixed batch of prompts as users send them
        {"name": "prompts ragged", "kind": "prompt", "seqs": 6, "median": 1024, "sigma": 1.0,
         "hk": 2, "hv": 8, "delta": True, "raw": True, "qk_norm": True, "norm": False, "shape": 5},
        # the benchmark's prompts, 8 x 4096, with the layer's output norm
        {"name": "prompts long", "kind": "prompt", "seqs": 8, "median": 4096, "sigma": 0.0,
         "hk": 2, "hv": 8, "delta": True, "raw": True, "qk_norm": True, "norm": True, "shape": 6},
        # one long document: few rows, a long axis
        {"name": "prompt document", "kind": "prompt", "seqs": 1, "median": 32768, "sigma": 0.0,
         "hk": 2, "hv": 8, "delta": True, "raw": True, "qk_norm": True, "norm": False, "shape": 7},
        # a decay alone over all heads of a model on one GPU
        {"name": "prompts decay only", "kind": "prompt", "seqs": 3, "median": 700, "sigma": 0.5,
         "hk": 16, "hv": 64, "delta": False, "raw": False, "qk_norm": False, "norm": False,
         "shape": 8},
        # the conv of the short chat turn, and of the benchmark's prompts
        {"name": "conv short", "kind": "conv", "seqs": 1, "median": 77, "sigma": 0.0, "hk": 2,
         "hv": 8, "width": 3, "shape": 9},
        {"name": "conv long", "kind": "conv", "seqs": 8, "median": 4096, "sigma": 0.0, "hk": 2,
         "hv": 8, "width": 4, "shape": 10},
        # the output norm of a decode batch, and of the benchmark's prompts
        {"name": "norm decode", "kind": "norm", "tokens": 256, "heads": 8, "dim": 128, "shape": 11},
        {"name": "norm prompts", "kind": "norm", "tokens": 32768, "heads": 8, "dim": 128,
         "shape": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["step", "step", "step", "prompt", "prompt", "prompt", "prompt", "conv",
                       "norm"])
    shape = rng.randrange(1 << 20)
    hk, hv = rng.choice([(2, 8), (2, 8), (2, 8), (16, 64), (8, 8), (4, 8), (1, 4)])
    how = {"hk": hk, "hv": hv, "delta": rng.random() < 0.75, "raw": rng.random() < 0.7,
           "qk_norm": rng.random() < 0.8, "norm": rng.random() < 0.4}
    if kind == "step":
        return {"kind": kind, "batch": _log(rng, 1, 2048 // hv), **how, "shape": shape}
    if kind == "norm":
        heads, dim = rng.choice([(8, 128), (8, 128), (64, 128), (1, 64), (4, 256), (3, 200),
                                 (1, 1000), (1, 4096)])
        return {"kind": kind, "tokens": _log(rng, 1, (1 << 25) // (heads * dim)), "heads": heads,
                "dim": dim, "shape": shape}
    seqs = _log(rng, 1, 32)
    sigma = rng.choice([0.0, 0.5, 1.0])
    # a sequence is at most 4 medians long, and all of them the largest case's tokens
    median = _log(rng, 2, MOST // (hv * seqs * (4 if sigma and seqs > 1 else 1)))
    if kind == "conv":
        return {"kind": kind, "seqs": seqs, "median": median, "sigma": sigma, "hk": hk, "hv": hv,
                "width": rng.choice([3, 4]), "shape": shape}
    return {"kind": kind, "seqs": seqs, "median": median, "sigma": sigma, **how, "shape": shape}


# --- the workload's shape, from the case alone -------------------------------------------


def _lengths(case):
    n, g = case["seqs"], np.random.default_rng(case["shape"])
    x = case["median"] * np.exp(case["sigma"] * g.standard_normal(n))
    most = 4 * case["median"] if n > 1 else case["median"]
    return np.clip(np.rint(x), 1, most).astype(np.int64)


def _slots(case, n):
    """n distinct slots of a pool with a few more, in no order."""
    size = n + 3
    return size, np.random.default_rng(case["shape"] + 1).permutation(size)[:n].astype(np.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*size):
        return torch.randn(*size, generator=gen, device="cuda")

    def uniform(*size):
        return torch.rand(*size, generator=gen, device="cuda")

    silu = torch.nn.functional.silu
    st = {"case": case, "kind": case["kind"]}
    if case["kind"] == "norm":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        st["x"] = (0.2 * normal(t, h, d)).bfloat16()
        st["z"] = normal(t, h, d).bfloat16()
        st["weight"] = (1 + 0.1 * normal(d)).bfloat16()
        return st
    hk, hv = case["hk"], case["hv"]
    channels = (2 * hk + hv) * D
    if case["kind"] == "step":
        tokens = n = case["batch"]
    else:
        lens = _lengths(case)
        tokens, n = int(lens.sum()), len(lens)
        cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        st["cu"], st["longest"] = torch.from_numpy(cu).cuda(), int(lens.max())
    size, slots = _slots(case, n)
    st["slots"] = torch.from_numpy(slots).cuda()
    if case["kind"] == "conv":
        st["x"] = normal(tokens, channels).bfloat16()
        st["weight"] = (0.5 * normal(channels, 4)).bfloat16()
        st["conv"] = normal(size, channels, case["width"]).bfloat16()
        return st
    # q, k and v are views of the conv's output, as the layer has them
    mixed = silu(normal(tokens, channels))
    if not case["qk_norm"]:  # the caller has normalised q and k
        qk = mixed[:, :2 * hk * D].view(tokens, 2 * hk, D)
        qk /= (qk.square().sum(-1, keepdim=True) + L2_EPS).sqrt()
    mixed = mixed.bfloat16()
    st["q"] = mixed[:, :hk * D].view(tokens, hk, D)
    st["k"] = mixed[:, hk * D:2 * hk * D].view(tokens, hk, D)
    st["v"] = mixed[:, 2 * hk * D:].view(tokens, hv, D)
    if case["raw"]:
        # projections, and the usual range of initial decays: A in [1, 16], steps of 0.001 to 0.1
        st["g"] = normal(tokens, hv).bfloat16()
        st["beta"] = normal(tokens, hv).bfloat16()
        st["a_log"] = (1 + 15 * uniform(hv)).log()
        step = (math.log(1e-3) + math.log(100.0) * uniform(hv)).exp()
        st["dt_bias"] = step + torch.log(-torch.expm1(-step))
    else:
        st["g"] = -(0.001 + 0.5 * uniform(tokens, hv).square())
        st["beta"] = torch.sigmoid(normal(tokens, hv))
        st["a_log"] = st["dt_bias"] = None
    if not case["delta"]:
        st["beta"] = None
    st["z"] = normal(tokens, hv, D).bfloat16() if case["norm"] else None
    st["weight"] = (1 + 0.1 * normal(D)).bfloat16() if case["norm"] else None
    st["state"] = 0.1 * normal(size, hv, D, D)
    return st


# --- the framework's calls -----------------------------------------------------------------


def _own(st):
    from muserve_amd.kernels import linear_attention as la
    kind = st["kind"]
    if kind == "norm":
        return la.gated_rms_norm(st["x"], st["z"], st["weight"], EPS)
    if kind == "conv":
        out = la.causal_conv_prefill(st["x"], st["weight"], st["conv"], st["slots"], st["cu"])
        return out, st["conv"]
    more = {"a_log": st["a_log"], "dt_bias": st["dt_bias"], "qk_norm": st["case"]["qk_norm"],
            "z": st["z"], "norm_weight": st["weight"], "norm_eps": EPS}
    if kind == "step":
        out = la.linear_attn_decode(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"],
                                    st["slots"], **more)
    else:
        out = la.linear_attn_prefill(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"],
                                     st["slots"], st["cu"], max_seqlen=st["longest"], **more)
    return out, st["state"]


# --- the plain form ------------------------------------------------------------------------


def _silu(x):
    return x / (1 + torch.exp(-x))


def _gated_norm(x, z, w, eps=EPS):
    z = z.to(x.dtype)
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.to(x.dtype) * _silu(z)


def _inputs(st, dtype):
    """q, k, v, log decays and betas in `dtype`, q and k normalised and one for each value head."""
    q, k, v = (st[x].to(dtype) for x in "qkv")
    if st["case"]["qk_norm"]:
        q = q / (q.square().sum(-1, keepdim=True) + L2_EPS).sqrt()
        k = k / (k.square().sum(-1, keepdim=True) + L2_EPS).sqrt()
    of = torch.arange(v.shape[1], device=v.device) // (v.shape[1] // k.shape[1])
    g, beta = st["g"].to(dtype), st["beta"]
    if st["case"]["raw"]:
        x = g + st["dt_bias"].to(dtype)
        softplus = x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))
        g = -torch.exp(st["a_log"].to(dtype)) * softplus
    if beta is not None:
        beta = beta.to(dtype)
        if st["case"]["raw"]:
            beta = 1 / (1 + torch.exp(-beta))
    return q[:, of], k[:, of], v, g, beta


def _step(st):
    q, k, v, g, beta = _inputs(st, torch.float32)
    at = st["slots"].long()
    s = st["state"][at] * torch.exp(g)[..., None, None]
    u = v if beta is None else beta[..., None] * (v - (s * k[:, :, None, :]).sum(-1))
    s = s + u[..., None] * k[:, :, None, :]
    st["state"][at] = s
    o = (s * q[:, :, None, :]).sum(-1) * D ** -0.5
    if st["z"] is not None:
        o = _gated_norm(o, st["z"], st["weight"])
    return o.bfloat16(), st["state"]


def _rows(st):
    """Packed rows by sequence: [sequences, longest] indices, and which of them exist."""
    cu = st["cu"].long()
    lens = cu[1:] - cu[:-1]
    pos = torch.arange(-(-st["longest"] // CHUNK) * CHUNK, device=cu.device)
    there = pos < lens[:, None]
    return torch.where(there, cu[:-1, None] + pos, torch.zeros_like(pos)), there


def _prompt(st):
    q, k, v, g, beta = _inputs(st, torch.float32)
    rows, there = _rows(st)
    n, length = rows.shape

    def chunks(x):  # [tokens, heads, ...] -> [sequences, heads, chunks, CHUNK, ...], zeros outside
        x = x[rows] * there.view(n, length, *[1] * (x.dim() - 1))
        return x.transpose(1, 2).unflatten(2, (-1, CHUNK))

    q, k, v = chunks(q), chunks(k), chunks(v)
    run = chunks(g.double()).cumsum(-1)
    i = torch.arange(CHUNK, device=q.device)
    below = i[:, None] >= i
    far = torch.where(below, run[..., :, None] - run[..., None, :], -math.inf)
    decay = torch.exp(far.float())                              # e^(G_i - G_j), j <= i
    p = torch.matmul(q, k.transpose(-1, -2).contiguous()) * decay
    head = torch.exp(run.float())[..., None]                    # e^G
    tail = torch.exp((run[..., -1:] - run).float())[..., None]  # e^(G_C - G)
    if beta is None:
        t = None
    else:
        b = chunks(beta)
        a = torch.matmul(k, k.transpose(-1, -2).contiguous()) * decay * b[..., None]
        t = torch.zeros_like(a)
        t[..., i, i] = 1
        for r in range(1, CHUNK):  # the unit lower triangle's inverse, row by row
            t[..., r, :r] = -torch.matmul(a[..., r:r + 1, :r], t[..., :r, :r]).squeeze(-2)
        t = t * b[..., None, :]
    at = st["slots"].long()
    s = st["state"][at].transpose(-1, -2).contiguous()          # [key, value]
    out = torch.empty_like(v)
    for c in range(v.shape[2]):
        kc = k[:, :, c]
        u = v[:, :, c]
        if t is not None:
            u = torch.matmul(t[:, :, c], u - head[:, :, c] * torch.matmul(kc, s))
        out[:, :, c] = head[:, :, c] * torch.matmul(q[:, :, c], s) + torch.matmul(p[:, :, c], u)
        more = torch.matmul((kc * tail[:, :, c]).transpose(-1, -2).contiguous(), u)
        s = head[:, :, c, -1:] * s + more
    st["state"][at] = s.transpose(-1, -2)
    o = out.flatten(2, 3).transpose(1, 2)[there] * D ** -0.5
    if st["z"] is not None:
        o = _gated_norm(o, st["z"], st["weight"])
    return o.bfloat16(), st["state"]


def _conv(st):
    rows, there = _rows(st)
    taps = st["weight"].float()
    width = st["conv"].shape[-1]
    at = st["slots"].long()
    x = torch.where(there[..., None], st["x"][rows], 0)
    x = torch.cat([st["conv"][at].transpose(1, 2), x], 1)      # the last `width` inputs first
    length = rows.shape[1]
    first = width - 3
    f = x.float()
    y = sum(taps[:, j] * f[:, first + j:first + j + length] for j in range(4))
    lens = there.sum(1)
    last = lens[:, None] + torch.arange(width, device=x.device)
    st["conv"][at] = torch.take_along_dim(x, last[..., None], 1).transpose(1, 2)
    return _silu(y)[there].bfloat16(), st["conv"]


def run(st):
    if own:
        return _own(st)
    if st["kind"] == "step":
        return _step(st)
    if st["kind"] == "prompt":
        return _prompt(st)
    if st["kind"] == "conv":
        return _conv(st)
    return _gated_norm(st["x"].float(), st["z"].float(), st["weight"].float()).bfloat16()


# --- what a pass cannot do without ----------------------------------------------------------


def work(case):
    if case["kind"] == "norm":
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 6 * values + 2 * case["dim"], "flops": 12 * values}
    hk, hv = case["hk"], case["hv"]
    channels = (2 * hk + hv) * D
    if case["kind"] == "conv":
        tokens, n = int(_lengths(case).sum()), case["seqs"]
        return {"bytes": 4 * tokens * channels + 4 * n * channels * case["width"] + 8 * channels,
                "flops": 12 * tokens * channels}
    tokens = n = case.get("batch", 0)
    if case["kind"] == "prompt":
        tokens, n = int(_lengths(case).sum()), case["seqs"]
    gate = (2 if case["raw"] else 4) * (2 if case["delta"] else 1)
    row = 2 * channels + 2 * hv * D * (2 if case["norm"] else 1) + gate * hv
    if case["kind"] == "step":
        flops = tokens * hv * D * D * (7 if case["delta"] else 5)
    else:
        # of a chunk and head: K S^T, Q S^T and U^T K over 128 x 128, the 64-term lower triangles
        # K K^T, Q K^T, T V and P U
        whole, low = (3, 4) if case["delta"] else (2, 2)
        flops = tokens * hv * 2 * D * (whole * D + low * CHUNK // 2)
    return {"bytes": tokens * row + 8 * n * hv * D * D, "flops": flops}


# --- the definition in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    double = torch.float64
    if case["kind"] == "norm":
        x, z = st["x"].to(double), st["z"].to(double)
        mean = (x * x).sum(-1, keepdim=True) / x.shape[-1]
        return st["weight"].to(double) * x * torch.rsqrt(mean + EPS) * z * torch.sigmoid(z)
    slots = st["slots"].tolist()
    if case["kind"] == "conv":
        cu, w, out = st["cu"].tolist(), st["weight"].to(double), []
        conv, width = st["conv"].to(double), case["width"]
        for b, slot in enumerate(slots):
            past = torch.cat([conv[slot].t(), st["x"][cu[b]:cu[b + 1]].to(double)])
            y = (past[width - 3:].unfold(0, 4, 1) * w).sum(-1)
            out.append(y * torch.sigmoid(y))
            conv[slot] = past[-width:].t()
        return torch.cat(out), conv
    steps = 1 if case["kind"] == "step" else st["longest"]
    if case["kind"] == "prompt" and steps * (1 + st["slots"].numel() * case["hv"] / 400) > 60000:
        return None  # the recurrence, token by token, takes too long
    q, k, v, g, beta = _inputs64(st)
    tokens, hv = g.shape
    n = len(slots)
    cu = torch.arange(n + 1, device=q.device) if steps == 1 and case["kind"] == "step" \
        else st["cu"].long()
    at = st["slots"].long()
    state = st["state"].to(double)
    s = state[at]
    out = torch.zeros(tokens + 1, hv, D, dtype=double, device=q.device)
    for t in range(steps):
        row = cu[:-1] + t
        there = row < cu[1:]
        r = torch.where(there, row, 0)
        kt, vt, qt = k[r], v[r], q[r]
        new = s * torch.exp(g[r])[:, :, None, None]
        u = vt if beta is None else beta[r][..., None] * (vt - torch.einsum("bhvk,bhk->bhv", new, kt))
        new = new + torch.einsum("bhv,bhk->bhvk", u, kt)
        s = torch.where(there[:, None, None, None], new, s)
        out[torch.where(there, row, tokens)] = torch.einsum("bhvk,bhk->bhv", new, qt)
    state[at] = s
    o = out[:tokens] / math.sqrt(D)
    if st["z"] is not None:
        z = st["z"].to(double)
        mean = (o * o).sum(-1, keepdim=True) / D
        o = st["weight"].to(double) * o * torch.rsqrt(mean + EPS) * z * torch.sigmoid(z)
    return o, state


def _inputs64(st):
    case = st["case"]
    q, k, v, g = (st[x].to(torch.float64) for x in "qkvg")
    if case["qk_norm"]:
        q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + L2_EPS)
        k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + L2_EPS)
    share = v.shape[1] // k.shape[1]
    q, k = q.repeat_interleave(share, 1), k.repeat_interleave(share, 1)
    beta = None if st["beta"] is None else st["beta"].to(torch.float64)
    if case["raw"]:
        g = -st["a_log"].to(torch.float64).exp() * torch.nn.functional.softplus(
            g + st["dt_bias"].to(torch.float64), threshold=1000)
        beta = None if beta is None else torch.sigmoid(beta)
    return q, k, v, g, beta
