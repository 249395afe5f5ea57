"""Linear attention over the state pool, the prompt conv and the gated norm on
the GPU against the float64 oracle (bounds in tests/linear_util.py)."""
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels import linear_attention as la
from muserve_amd.state_pool import StatePool
from oracle import linear as ref
from tests import linear_util as lu
from tests.gpu_util import DEV, case

pytestmark = pytest.mark.gpu
D = 128


def step(x, slots, state, **more):
    q, k, v = lu.split(x["mixed"], x["hk"], x["hv"])
    return la.linear_attn_decode(q, k, v, x["g"], x["beta"], state, slots, **lu.keywords(x), **more)


def prompt(x, slots, cu, state, **more):
    q, k, v = lu.split(x["mixed"], x["hk"], x["hv"])
    return la.linear_attn_prefill(q, k, v, x["g"], x["beta"], state, slots, cu, **lu.keywords(x),
                                  **more)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


HOW = [dict(), dict(raw=False), dict(delta=False), dict(qk_norm=False, raw=False),
       dict(delta=False, raw=False, qk_norm=False)]


@pytest.mark.parametrize("how", HOW, ids=str)
@pytest.mark.parametrize("batch,hk,hv,norm", [(1, 2, 8, False), (5, 2, 8, True), (3, 4, 4, False),
                                              (2, 1, 7, True)])
def test_decode(batch, hk, hv, norm, how):
    case(f"linear attention decode, {batch} x {hk}/{hv} heads, norm {norm}, {how}")
    pool = batch + 2
    x = lu.inputs(batch + hv, batch, hk, hv, norm=norm, slots=pool, wide=True, **how)
    slots = torch.randperm(pool, generator=torch.Generator().manual_seed(batch))[:batch]
    gx = lu.on_gpu(x)
    out = step(gx, slots.to(DEV), gx["state"])
    torch.cuda.synchronize()
    la.check_errors(DEV)
    want = x["state"].double().clone()
    for b, s in enumerate(slots.tolist()):
        o, st, s_tol, o_tol = lu.want_sequence(x, slice(b, b + 1), x["state"][s])
        if norm:
            o, o_tol = lu.with_norm(x, slice(b, b + 1), o, o_tol)
        lu.close(out[b:b + 1], o, o_tol, f"request {b}")
        lu.close_state(gx["state"][s], st, s_tol, f"state of request {b}")
        want[s] = gx["state"][s].double().cpu()
    assert torch.equal(gx["state"].double().cpu(), want)  # the other slots as they were


def check_prompts(x, lens, slots, norm=False, first=0, **more):
    """Runs the packed prompts on the GPU and compares rows and states."""
    cu = [first]
    for n in lens:
        cu.append(cu[-1] + n)
    rows = x["mixed"].shape[0]
    gx = lu.on_gpu(x)
    out = torch.full((rows, x["hv"], D), 7.0, dtype=torch.bfloat16, device=DEV)
    got = prompt(gx, ints(slots), ints(cu), gx["state"], out=out, **more)
    assert got is out
    torch.cuda.synchronize()
    la.check_errors(DEV)
    for b, s in enumerate(slots):
        at = slice(cu[b], cu[b + 1])
        o, st, s_tol, o_tol = lu.want_sequence(x, at, x["state"][s])
        if norm:
            o, o_tol = lu.with_norm(x, at, o, o_tol, rounded=True)
        lu.close(out[at], o, o_tol, f"sequence {b} of {lens[b]}")
        lu.close_state(gx["state"][s], st, s_tol, f"state of sequence {b}")
    kept = [i for i in range(x["state"].shape[0]) if i not in slots or lens[slots.index(i)] == 0]
    assert torch.equal(gx["state"][kept].cpu(), x["state"][kept])
    assert (out[:first] == 7).all() and (out[cu[-1]:] == 7).all()  # rows of no sequence


LENS = [[1], [2, 0, 3], [63], [64], [65], [130, 1, 64, 0, 17], [0, 200], [191, 256]]


@pytest.mark.parametrize("how", HOW, ids=str)
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_prompts(lens, how):
    case(f"linear attention prompts {lens}, {how}")
    pool, total = len(lens) + 2, sum(lens) + 5
    hk, hv = (2, 8) if len(lens) % 2 else (3, 3)
    x = lu.inputs(sum(lens), total, hk, hv, slots=pool, **how)
    slots = torch.randperm(pool, generator=torch.Generator().manual_seed(len(lens))).tolist()
    check_prompts(x, lens, slots[:len(lens)], first=2)


@pytest.mark.parametrize("max_seqlen", [None, 1, 300])
def test_prompts_with_the_norm(max_seqlen):
    case(f"linear attention prompts with the output norm, max_seqlen {max_seqlen}")
    x = lu.inputs(11, 260, 2, 8, norm=True, slots=4)
    check_prompts(x, [70, 0, 180], [3, 1, 0], norm=True, first=4, max_seqlen=max_seqlen)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("what", ["v", "k", "q", "g", "beta", "big v", "large v", "larger v",
                                  "no decay left", "growth"])
def test_what_is_not_finite_reaches_later_tokens_only(what, delta):
    """An infinity or NaN of one token leaves the tokens before it, the other
    heads, value dims (for v) and sequences as they were without it."""
    case(f"linear attention prompts with {what} of one token, delta {delta}")
    if what == "beta" and not delta:
        return
    lens, at, hk, hv = [70, 130, 40], 70 + 64 + 21, 2, 8
    x = lu.inputs(5, 240, hk, hv, slots=3, raw=False, delta=delta)
    clean = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in x.items()}
    q, k, v = lu.split(x["mixed"], hk, hv)
    if what == "v":
        v[at, 5, 17], v[at, 5, 90] = float("inf"), float("nan")
    elif what == "k":
        k[at, 1, 3] = float("nan")
    elif what == "q":
        q[at, 1, 3] = float("inf")
    elif what == "g":
        x["g"][at, 5] = float("nan")
    elif what == "beta":
        x["beta"][at, 5] = float("nan")
    elif what == "big v":
        v[at, 5, 17] = 2.0 ** 100
    elif what == "large v":
        v[at, 5, 17] = 2.0 ** 24
    elif what == "larger v":
        v[at, 5, 17] = 2.0 ** 50
    elif what == "no decay left":  # everything before it is forgotten: still finite
        x["g"][at, 5] = -float("inf")
    elif what == "growth":
        x["g"][at, 5] = 60.0
    gx = lu.on_gpu(x)
    out = prompt(gx, ints([0, 1, 2]), ints([0, 70, 200, 240]), gx["state"])
    la.check_errors(DEV)
    assert torch.isfinite(out[:at].float()).all() and torch.isfinite(out[200:].float()).all()
    if what in ("no decay left", "growth"):
        assert torch.isfinite(out.float()).all()
    hit = [4, 5, 6, 7] if what in ("k", "q") else [5]
    for b, (r0, r1) in enumerate(((0, 70), (70, 200), (200, 240))):
        o, st, s_tol, o_tol = lu.want_sequence(clean, slice(r0, r1), clean["state"][b])
        for h in range(hv):
            to = min(r1, at) if h in hit else r1
            if to > r0:
                lu.close(out[r0:to, h], o[:to - r0, h], o_tol[:to - r0, h], f"{b} head {h}")
            if h not in hit or b != 1:
                lu.close_state(gx["state"][b, h:h + 1], st[h:h + 1], s_tol[h:h + 1], f"state {b}")
    got = out[at:200, 5].float()
    if what == "v":  # an infinite or NaN value stays in its value dim
        others = [i for i in range(D) if i not in (17, 90)]
        assert torch.isfinite(got[:, others]).all() and not torch.isfinite(got[:, 90]).any()
        assert not torch.isfinite(got[0, 17])
    elif what in ("k", "g", "beta"):
        assert got.isnan().all() and not torch.isfinite(gx["state"][1, 5]).any()
    elif what == "q":  # a query is its own token's
        assert not torch.isfinite(got[0]).any() and torch.isfinite(got[1:]).all()
    elif what in ("no decay left", "growth"):
        o, st, s_tol, o_tol = lu.want_sequence(x, slice(70, 200), x["state"][1])
        if what == "no decay left":
            lu.close(out[70:200], o, o_tol, what)
            lu.close_state(gx["state"][1], st, s_tol, what)
        else:  # e^60: sizes are relative to the state's own, about its largest
            want = st[5]
            assert float((gx["state"][1, 5].double().cpu() - want).norm() / want.norm()) < 1e-4


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("size", [dict(v=1e-4), dict(v=2.0 ** 40), dict(beta=1e-3), dict(q=1e-5),
                                  dict(q=1e4), dict(k=1e-5), dict(k=1e-2, v=1e3),
                                  dict(state=1e-6), dict(state=1e6), dict(state=0.0),
                                  dict(v=0.0), dict(first=1e-7), dict(first=0.0), dict(last=3e4)],
                         ids=str)
def test_sizes(size, delta):
    """Inputs far from 1, all of them or the first or last tokens' alone."""
    case(f"linear attention prompts with inputs of other sizes, {size}, delta {delta}")
    x = lu.inputs(12, 150, 2, 8, raw=False, delta=delta, qk_norm="q" not in size and "k" not in size)
    q, k, v = lu.split(x["mixed"], 2, 8)
    for name, f in size.items():
        if name in ("q", "k", "v"):
            {"q": q, "k": k, "v": v}[name].mul_(f)
        elif name == "first":
            v[:3] *= f
        elif name == "last":
            v[140:] *= f
        elif x[name] is not None:
            x[name] *= f
    check_prompts(x, [150], [0])


def test_strong_decays_keep_their_ratios():
    """Log decays of -50 a token next to ones of -0.01: sums far from 0 whose
    differences are small."""
    case("linear attention prompts under strong decays")
    x = lu.inputs(6, 200, 2, 8, raw=False, slots=1)
    gen = torch.Generator().manual_seed(1)
    strong = torch.rand(200, 8, generator=gen) < 0.3
    x["g"] = torch.where(strong, torch.full_like(x["g"], -50.0), x["g"] * 0.1)
    x["g"][100:110] = -3e38
    check_prompts(x, [200], [0])


def test_large_launches_run_their_heads_in_turn():
    """More images than one launch holds: key heads in turn, with each key head's
    share alone as the reference. Its walk may be cut otherwise: outputs differ by
    two roundings to bf16 (2^-8 relative each), states by what fp32 sums do."""
    case("linear attention prompts, 16/64 heads x 66000 tokens in several launches")
    T, hk, hv = 66000, 16, 64
    gen = torch.Generator(device=DEV).manual_seed(3)
    q, k = (torch.randn(T, hk, D, generator=gen, device=DEV).bfloat16() for _ in range(2))
    v = torch.randn(T, hv, D, generator=gen, device=DEV).bfloat16()
    g = -torch.rand(T, hv, generator=gen, device=DEV)
    beta = torch.rand(T, hv, generator=gen, device=DEV)
    state = torch.randn(2, hv, D, D, generator=gen, device=DEV)
    cu, at = ints([0, 40000, T]), ints([1, 0])
    want = state.clone()
    out = la.linear_attn_prefill(q, k, v, g, beta, state, at, cu, qk_norm=True)
    for kh in (0, 7, 15):
        vh = slice(4 * kh, 4 * kh + 4)
        st = want[:, vh].contiguous()
        some = la.linear_attn_prefill(q[:, kh:kh + 1].contiguous(), k[:, kh:kh + 1].contiguous(),
                                      v[:, vh].contiguous(), g[:, vh].contiguous(),
                                      beta[:, vh].contiguous(), st, at, cu, qk_norm=True)
        for got, ref_, tol in ((out[:, vh], some, 2.0 ** -7), (state[:, vh], st, 1e-5)):
            ref_ = ref_.double()
            assert (got.double() - ref_).norm() <= tol * ref_.norm()
    la.check_errors(DEV)


def test_prompt_in_pieces_and_steps():
    """A prompt in chunks and then token by token gives what one call gives."""
    case("linear attention prompt whole, in pieces, and step by step")
    x = lu.inputs(3, 150, 2, 8, slots=2)
    gx = lu.on_gpu(x)
    states = [gx["state"].clone() for _ in range(3)]
    one = ints([1])
    whole = prompt(gx, one, ints([0, 150]), states[0])
    rows = lambda a, b: {n: t[a:b] if n in ("mixed", "g", "beta") else t for n, t in gx.items()}  # noqa: E731
    parts = torch.cat([prompt(rows(a, b), one, ints([0, b - a]), states[1])
                       for a, b in ((0, 64), (64, 101), (101, 150))])
    steps = torch.cat([step(rows(t, t + 1), one, states[2]) for t in range(150)])
    la.check_errors(DEV)
    o, st, s_tol, o_tol = lu.want_sequence(x, slice(0, 150), x["state"][1])
    for name, got, state in (("whole", whole, states[0]), ("pieces", parts, states[1]),
                             ("steps", steps, states[2])):
        lu.close(got, o, o_tol, name)
        lu.close_state(state[1], st, s_tol, name)
        assert torch.equal(state[0].cpu(), x["state"][0])


def test_layer_through_the_pool():
    """A GDN layer as a serving step runs it: conv, linear attention with gates
    and norm, over prompts and then for three tokens, all in the pool's slots."""
    case("GDN layer through StatePool: prompts, then decode steps")
    hk, hv, lens, new = 2, 8, [97, 5, 33], 3
    C, layer, slots = (2 * hk + hv) * D, 1, [4, 0, 2]
    pool = StatePool(num_layers=2, num_slots=6, conv_shape=(C, 4), device=DEV)
    pool.check_unique = True
    pool.reset(slots)
    gen = torch.Generator().manual_seed(8)
    w = (0.5 * torch.randn(C, 1, 4, generator=gen)).bfloat16()
    conv = torch.zeros(6, C, 4, dtype=torch.bfloat16)
    state = torch.zeros(6, hv, D, D)
    total = sum(lens)
    x = lu.inputs(9, total + new * len(lens), hk, hv, norm=True)
    proj = torch.randn(total + new * len(lens), C, generator=gen).bfloat16()
    gx, gp, gw = lu.on_gpu(x), proj.to(DEV), w.to(DEV)
    cu = [0, 97, 102, 135]
    at = ints(slots)
    dev = lambda m: lu.split(m, hk, hv)  # noqa: E731

    def checked(mixed, want_mixed, mass, out, rows, b, prefill):
        # the conv against its oracle, then the layer on the values the GPU computed
        lu.close(mixed, want_mixed, 2.0 ** -20 * mass, "conv")
        y = {**x, "mixed": x["mixed"].clone()}
        y["mixed"][rows] = mixed.cpu()
        o, st, s_tol, o_tol = lu.want_sequence(y, rows, state[slots[b]])
        o, o_tol = lu.with_norm(y, rows, o, o_tol, rounded=prefill)
        lu.close(out, o, o_tol, "layer")
        lu.close_state(pool.state[layer, slots[b]], st, s_tol, "state")
        state[slots[b]] = pool.state[layer, slots[b]].cpu()

    mixed = pool.conv_prefill(layer, at, gp[:total], gw, ints(cu))
    how = {n: lu.keywords(gx)[n] for n in ("a_log", "dt_bias", "qk_norm", "norm_weight")}
    out = pool.linear_attn_prefill(layer, at, *dev(mixed), gx["g"][:total], gx["beta"][:total],
                                   ints(cu), z=gx["z"][:total], **how)
    torch.cuda.synchronize()
    pool.check_errors()
    for b in range(3):
        rows = slice(cu[b], cu[b + 1])
        want, mass = ref.conv_prompt(conv, slots[b], proj[rows], w.view(C, 4))
        checked(mixed[rows], want, mass, out[rows], rows, b, True)
    for t in range(new):
        r = slice(total + t * 3, total + t * 3 + 3)
        mixed = pool.conv_decode(layer, at, gp[r], gw)
        out = pool.linear_attn_decode(layer, at, *dev(mixed), gx["g"][r], gx["beta"][r],
                                      z=gx["z"][r], **how)
        torch.cuda.synchronize()
        pool.check_errors()
        for b in range(3):
            row = slice(r.start + b, r.start + b + 1)
            want, mass = ref.conv_prompt(conv, slots[b], proj[row], w.view(C, 4))
            checked(mixed[b:b + 1], want, mass, out[b:b + 1], row, b, False)
    assert torch.equal(pool.conv[layer].cpu(), conv)
    assert not pool.state[0].any() and not pool.conv[0].any()


@pytest.mark.parametrize("width,channels", [(3, 64), (4, 1536), (4, 520)])
@pytest.mark.parametrize("lens", [[1], [2, 0, 3], [4, 17, 64, 65, 1], [130]], ids=str)
def test_conv_prompts(lens, width, channels):
    case(f"prompt conv {lens}, {channels} channels, width {width}")
    gen = torch.Generator().manual_seed(sum(lens) + channels)
    n, total = len(lens), sum(lens) + 3
    conv = torch.randn(n + 2, channels, width, generator=gen).bfloat16()
    buf = torch.randn(total, channels + 16, generator=gen).bfloat16()
    x = buf[:, 8:8 + channels]
    w = (0.5 * torch.randn(channels, 4, generator=gen)).bfloat16()
    slots = torch.randperm(n + 2, generator=gen)[:n].tolist()
    cu = [1]
    for m in lens:
        cu.append(cu[-1] + m)
    gconv, gxx = conv.to(DEV), buf.to(DEV)[:, 8:8 + channels]
    out = torch.full((total, channels), 7.0, dtype=torch.bfloat16, device=DEV)
    la.causal_conv_prefill(gxx, w.to(DEV), gconv, ints(slots), ints(cu), out=out)
    torch.cuda.synchronize()
    la.check_errors(DEV)
    for b, s in enumerate(slots):
        rows = slice(cu[b], cu[b + 1])
        want, mass = ref.conv_prompt(conv, s, x[rows], w)
        # fp32 sums of 4 products and the silu: 2^-20 of the products' size
        lu.close(out[rows], want, 2.0 ** -20 * mass, f"sequence {b}")
    assert torch.equal(gconv.cpu().view(torch.int16), conv.view(torch.int16))
    assert (out[:1] == 7).all() and (out[cu[-1]:] == 7).all()


@pytest.mark.parametrize("tokens,heads,dim", [(1, 1, 8), (3, 2, 64), (5, 8, 128), (2, 3, 200),
                                              (7, 1, 512), (2, 1, 1000), (3, 1, 2048),
                                              (2, 2, 4096), (1000, 8, 128)])
def test_gated_norm(tokens, heads, dim):
    case(f"gated norm {tokens} x {heads} x {dim}")
    gen = torch.Generator().manual_seed(tokens + dim)
    x = (3 * torch.randn(tokens, heads, dim, generator=gen)).bfloat16()
    x[0] = 0
    zbuf = torch.randn(tokens, heads * dim + 8, generator=gen).bfloat16()
    for dtype in (torch.bfloat16, torch.float32):
        w = (1 + torch.randn(dim, generator=gen)).to(dtype)
        gz = zbuf.to(DEV)[:, :heads * dim].view(tokens, heads, dim)
        gx = x.to(DEV)
        out = la.gated_rms_norm(gx, gz, w.to(DEV), 1e-5)
        want = ref.gated_norm(x, zbuf[:, :heads * dim].view(tokens, heads, dim), w, 1e-5)
        # a sum of dim squares (positive: relative error sqrt(dim) 2^-24), a
        # root, a division, an exponential and a few products: 64 roundings
        lu.close(out, want, (64 + dim ** 0.5) * lu.U32 * want.abs(), str(dtype))
        la.gated_rms_norm(gx, gz, w.to(DEV), 1e-5, out=gx)  # in place
        assert torch.equal(gx, out)
    flat = la.gated_rms_norm(x[:, 0].contiguous().to(DEV), gz[:, 0].contiguous(), w.to(DEV), 1e-5)
    assert torch.equal(flat, out[:, 0])


def test_bad_slots_and_offsets():
    case("linear attention and conv: slots outside the pool, offsets that do not hold together")
    x = lu.inputs(4, 90, 2, 8, norm=True, slots=3)
    gx = lu.on_gpu(x)
    small = {n: t[:2] if n in ("mixed", "g", "beta", "z") else t for n, t in gx.items()}
    out = step(small, ints([3, 1]), gx["state"])
    with pytest.raises(_lib.MkvDeviceError, match="state-pool slot"):
        la.check_errors(DEV)
    assert not out[0].any() and out[1].any()
    assert torch.equal(gx["state"][[0, 2]].cpu(), x["state"][[0, 2]])
    gx = lu.on_gpu(x)
    out = prompt(gx, ints([-1, 2]), ints([0, 80, 90]), gx["state"])
    with pytest.raises(_lib.MkvDeviceError, match="state-pool slot"):
        la.check_errors(DEV)
    assert not out[:80].any() and out[80:].any()
    assert torch.equal(gx["state"][:2].cpu(), x["state"][:2])
    gx = lu.on_gpu(x)
    conv = torch.randn(3, 64, 4, device=DEV).bfloat16()
    rows = torch.randn(90, 64, device=DEV).bfloat16()
    w = torch.randn(64, 4, device=DEV).bfloat16()
    kept = conv.clone()
    for cu in ([0, 95, 90], [-3, 10, 90], [0, 40, 20], [0, 10, 91]):
        out = torch.full((90, 8, D), 7.0, dtype=torch.bfloat16, device=DEV)
        prompt(gx, ints([0, 1]), ints(cu), gx["state"], out=out)
        with pytest.raises(_lib.MkvDeviceError, match="inconsistent offsets"):
            la.check_errors(DEV)
        assert (out == 7).all() and torch.equal(gx["state"].cpu(), x["state"])
        y = torch.full((90, 64), 7.0, dtype=torch.bfloat16, device=DEV)
        la.causal_conv_prefill(rows, w, conv, ints([0, 1]), ints(cu), out=y)
        with pytest.raises(_lib.MkvDeviceError, match="inconsistent offsets"):
            la.check_errors(DEV)
        assert (y == 7).all() and torch.equal(conv, kept)
    y = la.causal_conv_prefill(rows, w, conv, ints([9, 1]), ints([0, 40, 90]))
    with pytest.raises(_lib.MkvDeviceError, match="state-pool slot"):
        la.check_errors(DEV)
    assert not y[:40].any() and y[40:].any() and torch.equal(conv[[0, 2]], kept[[0, 2]])


def test_duplicate_slots_are_reported_when_checked():
    case("linear attention through the pool: a repeated slot under the duplicate check")
    pool = StatePool(num_layers=1, num_slots=4, state_shape=(8, 128, 128), conv_shape=(64, 4),
                     device=DEV)
    pool.check_unique = True
    x = lu.on_gpu(lu.inputs(2, 2, 2, 8))
    q, k, v = lu.split(x["mixed"], 2, 8)
    pool.linear_attn_decode(0, ints([1, 3]), q, k, v, x["g"], x["beta"])
    pool.check_errors()
    with pytest.raises(IndexError):
        pool.linear_attn_decode(1, ints([1, 3]), q, k, v, x["g"], x["beta"])
    pool._unique.run(ints([1, 1]), pool._errors)
    with pytest.raises(_lib.MkvDeviceError, match="more than once"):
        pool.check_errors()


def test_argument_errors():
    case("linear attention: refused arguments")
    x = lu.on_gpu(lu.inputs(2, 4, 2, 8, norm=True, slots=5))
    q, k, v = lu.split(x["mixed"], 2, 8)
    g, b, st, sl, z, w = x["g"], x["beta"], x["state"], ints([0, 1, 2, 3]), x["z"], x["w"]
    dec, pre, cu = la.linear_attn_decode, la.linear_attn_prefill, ints([0, 1, 2, 3, 4])
    with pytest.raises(TypeError):
        dec(q.float(), k, v, g, b, st, sl)
    with pytest.raises(TypeError):
        dec(q, k, v, g.double(), b, st, sl)
    with pytest.raises(TypeError):
        dec(q, k, v, g, b.float(), st, sl)
    for bad in ((q[:3], k, v, g, b, st, sl), (q, k, v, g[:3], b, st, sl), (q, k, v, g, b, st, sl[:3]),
                (q, k, v[:, :7], g, b, st, sl), (q, k, v, g, b, st.double(), sl),
                (q, k, v, g, b, st[..., :64], sl), (q, k, v.transpose(1, 2), g, b, st, sl),
                (q, k[:, :1].expand(4, 2, D), v, g, b, st, sl), (q, k, v, g, b, st, sl.float())):
        with pytest.raises((ValueError, TypeError)):
            dec(*bad)
    for more in (dict(z=z), dict(norm_weight=w), dict(z=z[:3], norm_weight=w),
                 dict(z=z, norm_weight=w[:64]), dict(z=z, norm_weight=w.half()),
                 dict(a_log=x["a_log"]), dict(a_log=x["a_log"].double(), dt_bias=x["dt_bias"]),
                 dict(out=torch.empty(4, 8, 64, device=DEV).bfloat16())):
        with pytest.raises((ValueError, TypeError)):
            dec(q, k, v, g, b, st, sl, **more)
    with pytest.raises(ValueError):
        pre(q, k, v, g, b, st, sl, cu[:4])
    with pytest.raises(ValueError):
        pre(q, k, v, g, b, st, sl, cu, max_seqlen=-1)
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        dec(q, k, v, g, b, st.cpu(), sl)
    y = torch.zeros(4, 64, device=DEV).bfloat16()
    cw, cs = torch.zeros(64, 4, device=DEV).bfloat16(), torch.zeros(5, 64, 4, device=DEV).bfloat16()
    for bad in ((y.float(), cw, cs, sl, cu), (y, cw[:32], cs, sl, cu), (y[:, :32], cw, cs, sl, cu),
                (y, cw, cs, sl, cu[:2])):
        with pytest.raises((ValueError, TypeError)):
            la.causal_conv_prefill(*bad)
    with pytest.raises(ValueError, match="out must not be x"):
        la.causal_conv_prefill(y, cw, cs, sl, cu, out=y)
    for bad in ((z, z[:3], w), (z.float(), z, w), (z, z, w[:64]), (z[..., :60], z[..., :60], w[:60])):
        with pytest.raises((ValueError, TypeError)):
            la.gated_rms_norm(*bad)
    la.check_errors(DEV)
