"""Timed cases of an attention layer's operators around a KV pool on one GPU:

* ``rope``: the norm of each query and key head with the rotation by its position;
* ``rope append``: the same in one pass with the paged append of K and V (16-bit pools);
* ``window``: a pool held in 4 bits: the append of a prefill chunk, and the sequences' windows
  read back in bf16, as chunked prefill needs them;
* ``decode``: one query token per sequence over the 4-bit pool.

A 4-bit row of a token and head of 256 is 136 bytes: 128 bytes of e2m1 codes (the even dim in the
low half), then one e8m0 scale for every 32 dims: the least power of two 2^e with max |x| <= 7 2^e.

With ``own`` unset ``run`` computes the operators with elementary torch operations in fp32 (angles
in fp64), rounded once at the end; with ``own`` set it calls the package. Lengths, pages and slots
come from the case; the seed makes the values.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
D4 = 256                 # head dim of a 4-bit pool
ROW = D4 // 2 + D4 // 32  # bytes of a row of it
EPS = 1e-6
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_ROPE = 32768 * 5 * 256   # values of the largest rope case
MOST_WINDOW = 65536           # tokens x heads of the largest windows
MOST_DECODE = 1 << 20         # tokens x heads of a drawn decode case


def listed():
    return [
        # one interactive user's decode step on one rank of eight: latency and launches
        {"name": "rope one user", "kind": "rope", "tokens": 1, "hq": 4, "hk": 1, "dim": 256,
         "rot": 64, "style": "half", "type": "bf16", "gate": True, "far": 262144, "shape": 1},
        # the serving loop's full decode batch
        {"name": "rope decode batch", "kind": "rope", "tokens": 256, "hq": 4, "hk": 1, "dim": 256,
         "rot": 64, "style": "half", "type": "bf16", "gate": True, "far": 32768, "shape": 2},
        # the benchmark's prompts, 8 x 4096
        {"name": "rope prompts", "kind": "rope", "tokens": 32768, "hq": 4, "hk": 1, "dim": 256,
         "rot": 64, "style": "half", "type": "bf16", "gate": True, "far": 4096, "shape": 3},
        # another model's heads: every dim rotated in neighbouring pairs, an odd number of tokens
        {"name": "rope other heads", "kind": "rope", "tokens": 1021, "hq": 12, "hk": 3, "dim": 128,
         "rot": 128, "style": "pairs", "type": "fp16", "gate": False, "far": 32768, "shape": 4},
        # a decode batch's K and V straight into the pool, a page of its own for each
        {"name": "rope append decode batch", "kind": "rope append", "tokens": 256, "seqs": 256,
         "hq": 4, "hk": 1, "dim": 256, "rot": 64, "style": "half", "type": "bf16", "gate": True,
         "far": 32768, "shape": 5},
        # a step's prefill budget of 4096 tokens from a few requests
        {"name": "rope append chunk", "kind": "rope append", "tokens": 4096, "seqs": 3, "hq": 4,
         "hk": 1, "dim": 256, "rot": 64, "style": "half", "type": "bf16", "gate": True,
         "far": 32768, "shape": 6},
        # a short prompt into a 4-bit pool and its window
        {"name": "window short", "kind": "window", "seqs": 1, "chunk": 77, "prefix": 0, "hk": 1,
         "shape": 7},
        # two heads, chunks behind prefixes that end inside a page
        {"name": "window two heads", "kind": "window", "seqs": 3, "chunk": 333, "prefix": 1001,
         "hk": 2, "shape": 8},
        # the chunked-prefill benchmark's windows: chunks of 2048 in windows of 8192
        {"name": "window chunks", "kind": "window", "seqs": 8, "chunk": 2048, "prefix": 6144,
         "hk": 1, "shape": 9},
        # one interactive user
        {"name": "decode one user", "kind": "decode", "seqs": 1, "median": 2000, "sigma": 0.0,
         "hq": 4, "hk": 1, "shape": 10},
        # the decode benchmark's batch: 256 sequences, median 4096, at most 32768
        {"name": "decode full batch", "kind": "decode", "seqs": 256, "median": 4096, "sigma": 1.0,
         "hq": 4, "hk": 1, "shape": 11},
        # two long documents on two KV heads
        {"name": "decode documents", "kind": "decode", "seqs": 2, "median": 131072, "sigma": 0.0,
         "hq": 16, "hk": 2, "shape": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "rope append", "rope append", "window", "window", "decode",
                       "decode", "decode"])
    shape = rng.randrange(1 << 20)
    if kind.startswith("rope"):
        hq, hk, dim = rng.choice([(4, 1, 256), (4, 1, 256), (8, 2, 256), (32, 2, 256), (12, 3, 128),
                                  (16, 8, 128), (9, 3, 64), (1, 1, 64), (5, 5, 128)])
        rot = rng.choice([dim, dim // 2, dim // 4, 48])
        tokens = _log(rng, 1, MOST_ROPE // ((hq + hk) * dim))
        case = {"kind": kind, "tokens": tokens, "hq": hq, "hk": hk, "dim": dim, "rot": rot,
                "style": rng.choice(["half", "half", "pairs"]),
                "type": rng.choice(["bf16", "bf16", "fp16"]), "gate": rng.random() < 0.5,
                "far": _log(rng, 256, 262144), "shape": shape}
        if kind == "rope append":
            case["seqs"] = _log(rng, 1, min(tokens, 256))
        return case
    if kind == "window":
        seqs, hk = _log(rng, 1, 16), rng.choice([1, 1, 2, 3])
        window = _log(rng, 2, MOST_WINDOW // (seqs * hk))
        chunk = _log(rng, 1, window)
        return {"kind": kind, "seqs": seqs, "chunk": chunk, "prefix": window - chunk, "hk": hk,
                "shape": shape}
    hq, hk = rng.choice([(4, 1), (4, 1), (4, 1), (8, 1), (8, 2), (16, 2), (2, 1), (3, 3)])
    seqs = _log(rng, 1, 256)
    sigma = rng.choice([0.0, 0.5, 1.0])
    most = MOST_DECODE // (hk * seqs * (4 if sigma and seqs > 1 else 1))
    return {"kind": kind, "seqs": seqs, "median": _log(rng, 1, min(most, 131072)), "sigma": sigma,
            "hq": hq, "hk": hk, "shape": shape}


# --- the workload's shape, from the case alone -------------------------------------------


def _lengths(case):
    """Cached tokens of each sequence of a decode case."""
    n, g = case["seqs"], np.random.default_rng(case["shape"])
    x = case["median"] * np.exp(case["sigma"] * g.standard_normal(n))
    most = min(8 * case["median"], 32768) if case["sigma"] else case["median"]
    return np.clip(np.rint(x), 1, most).astype(np.int64)


def _tables(case, lens):
    """Block tables [n, widest] of pages in no order, and the pool's pages (a few more)."""
    pages = -(-lens // PAGE)
    total = int(pages.sum())
    order = np.random.default_rng(case["shape"] + 1).permutation(total + 3)[:total]
    tables = np.zeros((len(lens), int(pages.max())), dtype=np.int64)
    tables[np.arange(tables.shape[1]) < pages[:, None]] = order
    return tables, total + 3


def _split(total, n):
    """total tokens over n sequences, as even as they go."""
    return np.full(n, total // n) + (np.arange(n) < total % n)


def _slots(tables, starts, counts):
    """Slots of `counts` tokens from position `starts` of each sequence, and their positions."""
    seq = np.repeat(np.arange(len(counts)), counts)
    pos = np.arange(int(counts.sum())) - np.repeat(np.cumsum(counts) - counts - starts, counts)
    return tables[seq, pos // PAGE] * PAGE + pos % PAGE, pos


def _handle(pages, heads, dim, dtype):
    """The framework's pool, as a program keeps it."""
    if own:
        from muserve_amd.kv_cache import PagedKVCache
        return PagedKVCache(pages, num_layers=1, kv_heads=heads, head_dim=dim, dtype=dtype,
                            device="cuda:0", verbose=False)
    return None


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*size):
        return torch.randn(*size, generator=gen, device="cuda")

    kind, hk = case["kind"], case["hk"]
    st = {"case": case, "kind": kind}
    shape = np.random.default_rng(case["shape"])
    if kind.startswith("rope"):
        t, hq, dim = case["tokens"], case["hq"], case["dim"]
        dtype = torch.bfloat16 if case["type"] == "bf16" else torch.float16
        # views of one projection's output; a gate beside each query head where the layer has one
        wide = 2 * dim if case["gate"] else dim
        x = (3 * normal(t, hq * wide + 2 * hk * dim)).to(dtype)
        st["q"] = x[:, :hq * wide].unflatten(1, (hq, wide))[..., :dim]
        st["k"] = x[:, hq * wide:hq * wide + hk * dim].unflatten(1, (hk, dim))
        st["v"] = x[:, hq * wide + hk * dim:].unflatten(1, (hk, dim))
        st["q_weight"] = (0.1 * normal(dim)).to(dtype)   # around 1 once 1 is added
        st["k_weight"] = (0.1 * normal(dim)).to(dtype)
        i = torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64)
        st["inv_freq"] = (1e7 ** (-i / case["rot"])).float()
        if kind == "rope":
            pos = shape.integers(0, case["far"], t)
        else:
            counts = _split(t, case["seqs"])
            starts = shape.integers(0, PAGE, case["seqs"])
            tables, pages = _tables(case, starts + counts)
            slots, pos = _slots(tables, starts, counts)
            pos = pos + case["far"] // PAGE * PAGE - PAGE  # (pages in front are not in this pool)
            st["slots"] = torch.from_numpy(slots).cuda()
            st["cache"] = _handle(pages, hk, dim, dtype)
            st["pool"] = torch.empty(1, 2, pages, PAGE, hk, dim, dtype=dtype, device="cuda") \
                if st["cache"] is None else st["cache"].cache
            st["pool"].copy_(normal(*st["pool"].shape))
        st["positions"] = torch.from_numpy(pos).cuda()
        return st
    if kind == "window":
        n = case["seqs"]
        lens = np.full(n, case["prefix"] + case["chunk"])
        tables, pages = _tables(case, lens)
        slots, _ = _slots(tables, np.full(n, case["prefix"]), np.full(n, case["chunk"]))
        st["slots"] = torch.from_numpy(slots).cuda()
        st["k"] = normal(len(slots), hk, D4).bfloat16()
        st["v"] = normal(len(slots), hk, D4).bfloat16()
        st["cu"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)])).cuda()
        st["total"], st["longest"] = int(lens.sum()), int(lens.max())
        st["cache"] = _handle(pages, hk, D4, torch.float4_e2m1fn_x2)
        pool = torch.empty(1, 2, pages, PAGE, hk, ROW, dtype=torch.uint8, device="cuda") \
            if st["cache"] is None else st["cache"].cache
        pool[0, 0] = _quantise(normal(pages, PAGE, hk, D4).bfloat16().float())
        pool[0, 1] = _quantise(normal(pages, PAGE, hk, D4).bfloat16().float())
        st["pool"] = pool
    else:
        lens = _lengths(case)
        tables, pages = _tables(case, lens)
        st["q"] = normal(len(lens), 1, case["hq"], D4).bfloat16()
        st["k"], st["v"] = (_quantise(normal(pages, PAGE, hk, D4).bfloat16().float())
                            for _ in range(2))
    st["tables"] = torch.from_numpy(tables.astype(np.int32)).cuda()
    st["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
    return st


# --- the framework's calls -----------------------------------------------------------------


def _own(st):
    kind = st["kind"]
    if kind.startswith("rope"):
        how = {"zero_centered": True, "interleaved": st["case"]["style"] == "pairs"}
        if kind == "rope":
            from muserve_amd.kernels.rope import qk_norm_rope
            return qk_norm_rope(st["q"], st["k"], st["positions"], st["inv_freq"], st["q_weight"],
                                st["k_weight"], EPS, **how)
        q = st["cache"].append_rope(st["slots"], st["q"], st["k"], st["v"], 0, st["positions"],
                                    st["inv_freq"], st["q_weight"], st["k_weight"], EPS, **how)
        return q, st["cache"].cache
    if kind == "window":
        cache = st["cache"]
        cache.append(st["slots"], st["k"], st["v"], layer=0)
        out = tuple(torch.empty(st["total"], st["case"]["hk"], D4, dtype=torch.bfloat16,
                                device="cuda") for _ in range(2))
        return cache.gather(0, st["tables"], st["lens"], out_len=st["longest"], cu_out=st["cu"],
                            out=out)
    from muserve_amd.kernels.attention import attn_decode_fp4
    return attn_decode_fp4(st["q"], st["k"], st["v"], st["lens"], st["tables"])


# --- the plain form ------------------------------------------------------------------------


def _quantise(x):
    """fp32 [..., 256] of bf16 values -> 4-bit rows [..., 136]."""
    b = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))       # max = m 2^e, m in [1/2, 1)
    e = (e - 3 + (m > 0.875).int()).clamp(-120, 125)
    y = torch.ldexp(b, -e)
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5)
            + (a > 5)) + torch.signbit(y).byte() * 8
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return torch.cat([code[..., 0] + 16 * code[..., 1], (e + 127).byte().squeeze(-1)], -1)


def _values(rows, dtype=torch.float32):
    """4-bit rows [..., 136] -> the values [..., 256] that they stand for."""
    v = torch.tensor(VALUES, dtype=dtype, device=rows.device)
    v = torch.cat([v, -v])
    byte = torch.arange(256, device=rows.device)
    pairs = torch.stack([v[byte % 16], v[byte // 16]], -1)
    x = pairs[rows[..., :D4 // 2].int()].flatten(-2)
    scale = torch.ldexp(torch.ones((), dtype=dtype, device=rows.device),
                        rows[..., D4 // 2:].int() - 127)
    return (x.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _norm_rope(x, weight, st):
    x = x.float()
    x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * (1 + weight.float())
    angle = st["positions"].double()[:, None, None] * st["inv_freq"].double()
    c, s = angle.cos().float(), angle.sin().float()
    rot = st["case"]["rot"]
    turned = torch.empty_like(x)
    turned[..., rot:] = x[..., rot:]
    if st["case"]["style"] == "pairs":
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned[..., 0:rot:2], turned[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned[..., :rot // 2], turned[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return turned


def _rows_of(st):
    """[sequences, longest] slots of the block tables' tokens, and which of them exist."""
    pos = torch.arange(st["tables"].shape[1] * PAGE, device="cuda")
    slots = st["tables"].long()[:, pos // PAGE] * PAGE + pos % PAGE
    return slots, pos < st["lens"][:, None]


def _window(st):
    pool = st["pool"][0].flatten(1, 2)                       # [2, slots, heads, 136]
    pool[0, st["slots"]] = _quantise(st["k"].float())
    pool[1, st["slots"]] = _quantise(st["v"].float())
    slots, there = _rows_of(st)
    rows = slots[there]
    return _values(pool[0, rows]).bfloat16(), _values(pool[1, rows]).bfloat16()


def _decode(st):
    slots, there = _rows_of(st)
    n, length = slots.shape
    hk = st["k"].shape[2]
    q = st["q"].float().view(n, hk, -1, D4)
    # the tokens' values once, then padded to the longest sequence
    k, v = (torch.where(there[..., None, None], _values(x.flatten(0, 1))[slots * there], 0)
            for x in (st["k"], st["v"]))                     # [n, length, hk, 256]
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * D4 ** -0.5
    score = torch.where(there[:, None, None], score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p, v.transpose(1, 2).contiguous()).view(n, 1, -1, D4).bfloat16()


def run(st):
    if own:
        return _own(st)
    if st["kind"] == "window":
        return _window(st)
    if st["kind"] == "decode":
        return _decode(st)
    q = _norm_rope(st["q"], st["q_weight"], st).to(st["q"].dtype)
    k = _norm_rope(st["k"], st["k_weight"], st).to(st["k"].dtype)
    if st["kind"] == "rope":
        return q, k
    flat = st["pool"][0].flatten(1, 2)
    flat[0, st["slots"]], flat[1, st["slots"]] = k, st["v"]
    return q, st["pool"]


# --- what a pass cannot do without ----------------------------------------------------------


def work(case):
    kind, hk = case["kind"], case["hk"]
    if kind.startswith("rope"):
        t, dim = case["tokens"], case["dim"]
        turned = t * (case["hq"] + hk) * dim
        passed = t * hk * dim if kind == "rope append" else 0
        more = 8 * t * (2 if kind == "rope append" else 1) + 4 * dim + 2 * case["rot"]
        return {"bytes": 4 * (turned + passed) + more, "flops": 7 * turned}
    if kind == "window":
        chunk = case["seqs"] * case["chunk"] * hk
        window = case["seqs"] * (case["prefix"] + case["chunk"]) * hk
        return {"bytes": 2 * chunk * (2 * D4 + ROW) + 2 * window * (ROW + 2 * D4),
                "flops": 4 * D4 * chunk + 2 * D4 * window}
    tokens = int(_lengths(case).sum())
    return {"bytes": 2 * tokens * hk * ROW + 4 * case["seqs"] * case["hq"] * D4,
            "flops": 4 * tokens * case["hq"] * D4}


# --- the definition in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    double = torch.float64
    if case["kind"].startswith("rope"):
        half, pairs = case["rot"] // 2, case["style"] == "pairs"
        turn = torch.polar(torch.ones((), dtype=double, device="cuda"),
                           st["positions"].to(double)[:, None] * st["inv_freq"].to(double))

        def one(x, w):
            x = x.to(double)
            x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
            x = x * (w.to(double) + 1)
            head = x[..., :case["rot"]]
            z = head.unflatten(-1, (half, 2)) if pairs \
                else torch.stack([head[..., :half], head[..., half:]], -1)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn[:, None])
            z = z.flatten(-2) if pairs else torch.cat([z[..., 0], z[..., 1]], -1)
            return torch.cat([z, x[..., case["rot"]:]], -1)

        q, k = one(st["q"], st["q_weight"]), one(st["k"], st["k_weight"])
        if case["kind"] == "rope":
            return q, k
        pool = st["pool"].to(double)
        page, at = st["slots"] // PAGE, st["slots"] % PAGE
        pool[0, 0].index_put_((page, at), k)
        pool[0, 1].index_put_((page, at), st["v"].to(double))
        return q, pool
    lens = st["lens"].tolist()
    if case["kind"] == "window":
        out = []
        for plane, x in enumerate((st["k"], st["v"])):
            x = x.to(double).unflatten(-1, (8, 32))
            most = x.abs().amax(-1, keepdim=True)
            e = torch.floor(torch.log2(most)) - 2
            e = (e + (most > 7 * torch.exp2(e))).clamp(-120, 125)
            y = x / torch.exp2(e)
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1))) - 1)
            y = (torch.round(y / step) * step).clamp(-6, 6) * torch.exp2(e)
            pool = _values64(st["pool"][0, plane])
            pool.view(-1, case["hk"], D4)[st["slots"]] = y.flatten(-2)
            out.append(torch.cat([pool[t[:-(-n // PAGE)].long()].flatten(0, 1)[:n]
                                  for t, n in zip(st["tables"], lens)]))
        return tuple(out)
    out, group = [], case["hq"] // case["hk"]
    for b, n in enumerate(lens):
        pages = st["tables"][b, :-(-n // PAGE)].long()
        k = _values64(st["k"][pages]).flatten(0, 1)[:n]      # [n, hk, 256]
        v = _values64(st["v"][pages]).flatten(0, 1)[:n]
        rows = []
        for h in range(case["hq"]):
            score = (k[:, h // group] @ st["q"][b, 0, h].to(double)) / math.sqrt(D4)
            weight = torch.softmax(score, 0)
            rows.append((weight[:, None] * v[:, h // group]).sum(0))
        out.append(torch.stack(rows))
    return torch.stack(out)[:, None]


def _values64(rows):
    """4-bit rows, from their bits: a sign, two of exponent, one of mantissa; scales 2^(byte - 127)."""
    code = torch.stack([rows[..., :D4 // 2] & 15, rows[..., :D4 // 2] >> 4], -1).flatten(-2)
    sign, exp, man = code >> 3, (code >> 1) & 3, (code & 1).double()
    x = torch.where(exp == 0, man / 2, torch.exp2(exp.double() - 1) * (1 + man / 2))
    scale = torch.exp2(rows[..., D4 // 2:].double() - 127)
    return x * (1 - 2 * sign.double()) * scale.repeat_interleave(32, -1)
