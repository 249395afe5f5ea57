"""Linear attention over prompts with bounds for each value dim by itself, of what it
holds: it is as exact as its own size asks for, whatever its neighbours hold and it
has forgotten."""
import pytest
import torch

from oracle import linear as ref
from tests import linear_util as lu
from tests.gpu_util import DEV, case
from tests.test_gpu_linear_attention import ints, prompt

pytestmark = pytest.mark.gpu
D = 128


def want_by_dim(x, rows, state, scale=D ** -0.5):
    """The oracle on rows `rows` from `state`: outputs, final state, and the bounds of
    both for each value dim by itself (rows of S never meet).

    As in linear_util.want_sequence a token adds an error of sqrt(192) roundings of
    2^-24 of what the dim holds then, |S_n| + |u_n|, and sqrt(T) tokens add up; 8 of
    these leave nothing to chance. What a decay e^g shrinks takes its errors along, so
    the size an error is taken of is the largest so far with the decays since."""
    q, k, v = (t[rows] for t in lu.split(x["mixed"], x["hk"], x["hv"]))
    q, k, v = ref.normed(q, x["qk_norm"]), ref.normed(k, x["qk_norm"]), v.double()
    g, beta = ref.gates(x["g"][rows], None if x["beta"] is None else x["beta"][rows], x["a_log"],
                        x["dt_bias"])
    group = x["hv"] // x["hk"]
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    s = state.double().clone()
    size = s.norm(dim=-1)                                     # [Hv, Dv]
    out, o_tol = torch.zeros_like(v), torch.zeros_like(v)
    per = 8 * lu.U32 * (192 * v.shape[0]) ** 0.5
    for t in range(v.shape[0]):
        decay = g[t].exp()
        s = s * decay[:, None, None]
        u = v[t]
        if beta is not None:
            u = beta[t][:, None] * (u - (s * k[t][:, None, :]).sum(-1))
        s = s + u[:, :, None] * k[t][:, None, :]
        out[t] = scale * (s * q[t][:, None, :]).sum(-1)
        size = torch.maximum(size * decay[:, None], s.norm(dim=-1) + u.abs())
        o_tol[t] = 2 * abs(scale) * q[t].norm(dim=-1)[:, None] * per * size
    return out, s, per * size, o_tol


def check(x, T, **more):
    gx = lu.on_gpu(x)
    out = prompt(gx, ints([0]), ints([0, T]), gx["state"], **more)
    torch.cuda.synchronize()
    want, state, s_tol, o_tol = want_by_dim(x, slice(0, T), x["state"][0])
    lu.close(out, want, o_tol, "outputs")
    err = (gx["state"][0].double().cpu() - state).norm(dim=-1)
    bound = s_tol + 2.0 ** -140
    assert (err <= bound).all(), f"states: {float((err / bound).max()):.3g} times the bound"


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("qk_norm", [True, False])
@pytest.mark.parametrize("T", [9, 64, 150, 2600])
@pytest.mark.parametrize("spread", [12, 20, 40])
def test_value_dims_of_many_sizes(spread, T, qk_norm, delta):
    """One large dim among small ones, and dims of any size between."""
    case(f"linear attention, value dims 2^{spread} apart, {T} tokens, delta {delta}")
    hv = 4
    x = lu.inputs(70 + T, T, 2, hv, raw=False, delta=delta, qk_norm=qk_norm)
    gen = torch.Generator().manual_seed(spread)
    e = torch.randint(-spread // 2, spread // 2 + 1, (hv, D), generator=gen)
    e[0] = 0
    e[0, 5::16] = spread           # heads 0, 1: one of 16 dims unlike the others
    e[1] = spread // 2
    e[1, 3::16] = -spread // 2
    f = torch.ldexp(torch.ones(()), e)
    _, _, v = lu.split(x["mixed"], 2, hv)
    v.mul_(f.bfloat16())
    x["state"] *= f[None, :, :, None]
    check(x, T, max_seqlen=T)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("at", [3, 64 + 40])
def test_one_large_value(at, delta):
    """A value far above the others, in one dim of one token: its neighbours stay
    exact, at the token and after it."""
    case(f"linear attention, one large value at token {at}, delta {delta}")
    for size in (2.0 ** 12, 2.0 ** 20, 2.0 ** 50):
        x = lu.inputs(75, 200, 2, 4, raw=False, delta=delta)
        _, _, v = lu.split(x["mixed"], 2, 4)
        v[at, 1, 17] = size
        v[at, 2, 64:] *= size
        check(x, 200)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("T", [150, 2600])
@pytest.mark.parametrize("at,tokens,g", [(0, 1, -50.0), (30, 1, -50.0), (64, 1, -50.0),
                                         (127, 1, -30.0), (40, 30, -1.0), (100, 2, -3e38)])
def test_large_states_are_forgotten(at, tokens, g, T, delta):
    """States of 2^20 and 2^40 times the values, until a decay leaves nothing of them:
    what comes after is as exact as if they had not been."""
    case(f"linear attention, large states until {at} + {tokens} of {T} tokens, delta {delta}")
    x = lu.inputs(90, T, 2, 4, raw=False, delta=delta)
    x["g"] *= 0.02
    x["g"][at:at + tokens] = g
    x["state"][:, :2] *= 2.0 ** 20
    x["state"][:, 2] *= 2.0 ** 40
    x["state"][:, 3, ::2] *= 2.0 ** 20
    check(x, T, max_seqlen=T)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("at", [0, 20, 64, 90])
def test_large_values_are_forgotten(at, delta):
    """Values of 2^20 up to a strong decay, and of 1 after it."""
    case(f"linear attention, large values up to token {at}, delta {delta}")
    x = lu.inputs(91, 200, 2, 4, raw=False, delta=delta)
    _, _, v = lu.split(x["mixed"], 2, 4)
    v[:at + 1] *= 2.0 ** 20
    x["g"][at + 1] = -40.0
    check(x, 200)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("g", [-0.3, -2.0, -9.0])
def test_strong_decays_at_every_token(g, delta):
    case(f"linear attention, log decays near {g} at every token, delta {delta}")
    x = lu.inputs(92, 700, 2, 4, raw=False, delta=delta)
    x["g"] = g * (0.5 + torch.rand(700, 4, generator=torch.Generator().manual_seed(3)))
    check(x, 700)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("of", ["state", "values"])
def test_outputs_that_cancel(of, delta):
    """Queries of two elements whose products cancel to 2^-8 or less: an output's error
    is one of its terms, and these are not rounded to fewer bits than fp32 has."""
    case(f"linear attention, outputs that cancel, of the {of}, delta {delta}")
    T, hk, hv = 9, 2, 4
    x = lu.inputs(80, T, hk, hv, raw=False, delta=delta, qk_norm=False)
    gen = torch.Generator().manual_seed(81)
    q, k, v = lu.split(x["mixed"], hk, hv)
    x["g"] = x["g"][:, :1].expand(T, hv).contiguous()
    q.zero_()
    if of == "state":  # rows w_n a: the queries' keys are 0, 1, the others' from 64 on
        x["g"].zero_()
        k[..., :64] = 0
        a, w = torch.rand(D, generator=gen) + 1, torch.randn(hv, D, generator=gen)
        x["state"][0] = w[:, :, None] * a
        c = torch.rand(T, hk, generator=gen) + 0.5
        q[..., 0], q[..., 1] = c * a[1], -c * a[0]
    else:  # two writes that differ in sign, to keys 0 and 1, and decays between
        x["state"].zero_()
        k.zero_()
        k[0, :, 0] = k[1, :, 1] = 1
        v[1] = -v[0]
        v[2:] = 0
        if delta:
            x["beta"].fill_(1.0)
        decay = x["g"][1, 0].exp()
        c = torch.rand(T, hk, generator=gen) + 0.5
        q[2:, :, 0], q[2:, :, 1] = c[2:], c[2:] * decay
    check(x, T, max_seqlen=T)


@pytest.mark.parametrize("how", [dict(), dict(raw=False, qk_norm=False), dict(delta=False)], ids=str)
@pytest.mark.parametrize("T", [9, 30, 64, 150])
def test_outputs_by_value_dim(T, how):
    case(f"linear attention, bounds by value dim, {T} tokens, {how}")
    check(lu.inputs(82 + T, T, 2, 4, **how), T)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("T", [17, 30, 66, 131])
def test_small_values_at_the_end(T, delta):
    """The last one to three tokens of 2^-20 of the others, behind a decay that leaves
    nothing of those."""
    case(f"linear attention, small values at the end of {T} tokens, delta {delta}")
    x = lu.inputs(93, T, 2, 4, raw=False, delta=delta)
    last = T - T % 4
    assert 0 < T - last < 4
    _, _, v = lu.split(x["mixed"], 2, 4)
    v[last:] *= 2.0 ** -20
    x["g"][last] = -45.0
    x["state"] *= 0.1
    check(x, T)
