"""Packed prompts that do not start at row 0: the rows before the first sequence
and the slots of empty ones stay as they are (bounds in tests/linear_util.py)."""
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels import linear_attention as la
from muserve_amd.state_pool import StatePool
from oracle import linear as ref
from tests import linear_util as lu
from tests.gpu_util import DEV, case
from tests.test_gpu_linear_attention import check_prompts, ints, prompt

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("width", [3, 4])
@pytest.mark.parametrize("first", [15, 16, 17, 100, 255, 1000])
@pytest.mark.parametrize("lens", [[512], [0, 64, 3], [2] * 70, [0] * 66 + [40]],
                         ids=["one", "empty first", "70", "66 empty"])
def test_conv_behind_other_rows(lens, first, width):
    case(f"prompt conv of {len(lens)} sequences from row {first}, width {width}")
    gen = torch.Generator().manual_seed(first + len(lens))
    n, C, total = len(lens), 72, first + sum(lens) + 21
    conv = torch.randn(n, C, width, generator=gen).bfloat16()
    x = torch.randn(total, C, generator=gen).bfloat16()
    w = (0.5 * torch.randn(C, 4, generator=gen)).bfloat16()
    kept = torch.randn(total, C, generator=gen).bfloat16()
    cu = [first]
    for m in lens:
        cu.append(cu[-1] + m)
    gconv, out = conv.to(DEV), kept.to(DEV)
    la.causal_conv_prefill(x.to(DEV), w.to(DEV), gconv, ints(range(n)), ints(cu), out=out)
    torch.cuda.synchronize()
    la.check_errors(DEV)
    out = out.cpu()
    assert torch.equal(out[:first], kept[:first]) and torch.equal(out[cu[-1]:], kept[cu[-1]:])
    for b in range(n):
        rows = slice(cu[b], cu[b + 1])
        want, mass = ref.conv_prompt(conv, b, x[rows], w)
        lu.close(out[rows], want, 2.0 ** -20 * mass, f"sequence {b}")
    assert torch.equal(gconv.cpu(), conv)


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lens,first", [([2600], 1000), ([0, 2600], 512), ([0, 2600], 300),
                                        ([0, 2600] + [5, 0] * 34, 700)],
                         ids=["one", "empty first", "empty first, 300", "70"])
def test_long_prompts_behind_other_rows(lens, first, delta):
    """A first offset of more than a segment (these are walked in segments of 256
    tokens or a little more)."""
    case(f"linear attention over {len(lens)} prompts from row {first}, delta {delta}")
    x = lu.inputs(first, first + sum(lens) + 9, 1, 2, slots=len(lens), delta=delta)
    check_prompts(x, lens, list(range(len(lens)))[::-1], first=first, max_seqlen=max(lens))


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("lens", [[3000], [0, 3000]], ids=str)
def test_many_heads_behind_other_rows(lens, delta, norm):
    """32 heads (segments' ends by 16 waves): what the same rows give from row 0. The
    walk may be cut otherwise there: outputs differ by two roundings to bf16 of 2^-8
    each at most, states by what fp32 sums do (1e-5, in the norm over a head)."""
    case(f"linear attention of 32 heads from row 1100, {lens}, delta {delta}, norm {norm}")
    first, hk, hv, n = 1100, 2, 32, len(lens)
    total = first + sum(lens) + 7
    x = lu.on_gpu(lu.inputs(60, total, hk, hv, slots=n, delta=delta, norm=norm))
    cu = [0]
    for m in lens:
        cu.append(cu[-1] + m)
    kept = torch.randn(total, hv, D, device=DEV).bfloat16()
    out, states = kept.clone(), [x["state"].clone() for _ in range(2)]
    prompt(x, ints(range(n)), ints([first + c for c in cu]), states[0], out=out,
           max_seqlen=max(lens))
    some = {k: t[first:first + sum(lens)] if k in ("mixed", "g", "beta", "z") and t is not None
            else t for k, t in x.items()}
    want = prompt(some, ints(range(n)), ints(cu), states[1], max_seqlen=max(lens))
    torch.cuda.synchronize()
    la.check_errors(DEV)
    end = first + sum(lens)
    assert torch.equal(out[:first], kept[:first]) and torch.equal(out[end:], kept[end:])
    for b, m in enumerate(lens):
        if m == 0:
            assert torch.equal(states[0][b], x["state"][b])
    a, b = out[first:end].double(), want.double()
    assert ((a - b).abs() <= 2.0 ** -7 * b.norm(dim=-1, keepdim=True)).all()
    err = (states[0] - states[1]).double().flatten(2).norm(dim=2)
    assert (err <= 1e-5 * states[1].double().flatten(2).norm(dim=2)).all()


def test_prompts_of_a_step_behind_its_decode_rows():
    """A serving step as the planner packs it: decode tokens in the first rows, prompts
    behind them, both halves of a layer into one tensor each."""
    case("GDN layer over a step of 70 decode rows and two prompts")
    hk, hv, dec, lens = 2, 8, 70, [400, 33]
    C, total = (2 * hk + hv) * D, dec + sum(lens)
    x = lu.inputs(33, total, hk, hv, norm=True, slots=dec + 2)
    gen = torch.Generator().manual_seed(34)
    proj = torch.randn(total, C, generator=gen).bfloat16()
    w = (0.5 * torch.randn(C, 4, generator=gen)).bfloat16()
    pools = [StatePool(num_layers=1, num_slots=dec + 2, conv_shape=(C, 4), device=DEV)
             for _ in range(2)]
    for p in pools:
        p.state[0].copy_(x["state"])
        p.conv.copy_(torch.randn(p.conv.shape, generator=torch.Generator().manual_seed(35)))
    gx, gp, gw = lu.on_gpu(x), proj.to(DEV), w.to(DEV)
    cu = torch.tensor(list(range(dec + 1)) + [dec + lens[0], total], device=DEV)  # int64
    slots = ints(range(dec + 2))
    how = {n: lu.keywords(gx)[n] for n in ("a_log", "dt_bias", "qk_norm", "norm_weight")}

    def rows(at):
        return gx["g"][at], gx["beta"][at]

    # one tensor for the step: the decode half first, then the prompts into it
    mixed = torch.empty(total, C, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(total, hv, D, dtype=torch.bfloat16, device=DEV)
    at = slice(0, dec)
    mixed[at] = pools[0].conv_decode(0, slots[at], gp[at], gw)
    pools[0].conv_prefill(0, slots[dec:], gp, gw, cu[dec:], out=mixed)
    out[at] = pools[0].linear_attn_decode(0, slots[at], *lu.split(mixed[at], hk, hv), *rows(at),
                                          z=gx["z"][at], **how)
    pools[0].linear_attn_prefill(0, slots[dec:], *lu.split(mixed, hk, hv), gx["g"], gx["beta"],
                                 cu[dec:], z=gx["z"], out=out, max_seqlen=max(lens), **how)
    # the halves in tensors of their own
    m_dec = pools[1].conv_decode(0, slots[at], gp[at], gw)
    o_dec = pools[1].linear_attn_decode(0, slots[at], *lu.split(m_dec, hk, hv), *rows(at),
                                        z=gx["z"][at], **how)
    rest = slice(dec, total)
    m_pre = pools[1].conv_prefill(0, slots[dec:], gp[rest], gw, cu[dec:] - dec)
    o_pre = pools[1].linear_attn_prefill(0, slots[dec:], *lu.split(m_pre, hk, hv), *rows(rest),
                                         cu[dec:] - dec, z=gx["z"][rest], max_seqlen=max(lens),
                                         **how)
    torch.cuda.synchronize()
    for p in pools:
        p.check_errors()
    assert torch.equal(mixed[at], m_dec) and torch.equal(mixed[rest], m_pre)
    assert torch.equal(out[at], o_dec) and torch.equal(pools[0].conv, pools[1].conv)
    # (the prompt's walk may be cut otherwise, as above)
    a, b = out[rest].double(), o_pre.double()
    assert ((a - b).abs() <= 2.0 ** -7 * b.norm(dim=-1, keepdim=True)).all()
    err = (pools[0].state - pools[1].state).double().flatten(-2).norm(dim=-1)
    assert (err <= 1e-5 * pools[1].state.double().flatten(-2).norm(dim=-1)).all()


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("longest", [8, 70, 3000])
def test_bad_slots_and_offsets_in_every_form(longest, delta):
    """Token by token, in chunks and in segments (and 70 sequences of each)."""
    case(f"linear attention, bad slots and offsets, up to {longest} tokens, delta {delta}")
    for n in (2, 70):
        lens = [longest, 5] + [3] * (n - 2)
        total = sum(lens) + 6
        x = lu.on_gpu(lu.inputs(140, total, 1, 2, slots=n, delta=delta))
        cu = [1]
        for m in lens:
            cu.append(cu[-1] + m)
        kept = torch.randn(total, 2, D, device=DEV).bfloat16()
        for bad in (-1, n, 2 ** 31 - 1):
            state, out = x["state"].clone(), kept.clone()
            prompt(x, ints([bad, *range(1, n)]), ints(cu), state, out=out, max_seqlen=longest)
            with pytest.raises(_lib.MkvDeviceError, match="state-pool slot"):
                la.check_errors(DEV)
            assert not out[1:1 + longest].any() and out[1 + longest:cu[-1]].any()
            assert torch.equal(out[:1], kept[:1]) and torch.equal(out[cu[-1]:], kept[cu[-1]:])
            assert torch.equal(state[0], x["state"][0]) and not torch.equal(state[1], x["state"][1])
        for at, value in ((0, -1), (1, cu[2] + 1), (n, total + 1), (n // 2, 2 ** 31 - 1)):
            state, out, wrong = x["state"].clone(), kept.clone(), list(cu)
            wrong[at] = value
            prompt(x, ints(range(n)), ints(wrong), state, out=out, max_seqlen=longest)
            with pytest.raises(_lib.MkvDeviceError, match="inconsistent offsets"):
                la.check_errors(DEV)
            assert torch.equal(out, kept) and torch.equal(state, x["state"])


@pytest.mark.parametrize("call", ["linear_attn_decode", "linear_attn_prefill", "conv_prefill"])
def test_repeated_slots_through_the_calls(call):
    """Each in-place call reports a repeated slot where the pool checks (what the slots
    hold then is not said)."""
    case(f"StatePool.{call} with a repeated slot under the duplicate check")
    hk, hv, C = 2, 8, 64
    pool = StatePool(num_layers=1, num_slots=4, conv_shape=(C, 4), device=DEV)
    pool.check_unique = True
    x = lu.on_gpu(lu.inputs(2, 4, hk, hv))
    rows = torch.randn(4, C, device=DEV).bfloat16()
    w = torch.randn(C, 4, device=DEV).bfloat16()

    def run(slots):
        at = ints(slots)
        if call == "conv_prefill":
            pool.conv_prefill(0, at, rows, w, ints([0, 3, 4]))
        elif call == "linear_attn_prefill":
            pool.linear_attn_prefill(0, at, *lu.split(x["mixed"], hk, hv), x["g"], x["beta"],
                                     ints([0, 3, 4]))
        else:
            pool.linear_attn_decode(0, at, *lu.split(x["mixed"][:2], hk, hv), x["g"][:2],
                                    x["beta"][:2])
        pool.check_errors()

    run([1, 3])
    with pytest.raises(_lib.MkvDeviceError, match="more than once"):
        run([2, 2])
    run([2, 0])
