"""The output norm of prompts: taken of the fp32 outputs, rounded once, in every form
of the computation (bounds in tests/linear_util.py and by value dim)."""
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels import linear_attention as la
from tests import linear_util as lu
from tests.gpu_util import DEV, case
from tests.test_gpu_linear_attention import ints, prompt
from tests.test_gpu_linear_attention_sizes import want_by_dim

pytestmark = pytest.mark.gpu
D = 128


def check(x, lens, first=0, z=None, **more):
    cu = [first]
    for n in lens:
        cu.append(cu[-1] + n)
    gx = lu.on_gpu(x)
    if z is not None:
        gx["z"] = z
    kept = torch.randn(x["mixed"].shape[0], x["hv"], D, device=DEV).bfloat16()
    out = kept.clone()
    prompt(gx, ints(range(len(lens))), ints(cu), gx["state"], out=out, **more)
    torch.cuda.synchronize()
    la.check_errors(DEV)
    for b in range(len(lens)):
        rows = slice(cu[b], cu[b + 1])
        o, st, s_tol, o_tol = want_by_dim(x, rows, x["state"][b])
        y, y_tol = lu.with_norm(x, rows, o, o_tol)
        lu.close(out[rows], y, y_tol, f"sequence {b} of {lens[b]}")
        err = (gx["state"][b].double().cpu() - st).norm(dim=-1)
        assert (err <= s_tol + 2.0 ** -140).all()
    assert torch.equal(out[:first], kept[:first]) and torch.equal(out[cu[-1]:], kept[cu[-1]:])


@pytest.mark.parametrize("how", [dict(), dict(raw=False, qk_norm=False), dict(delta=False)], ids=str)
@pytest.mark.parametrize("lens,longest", [([1], 1), ([3, 0, 8], 8), ([9], 9), ([64], 64),
                                          ([130, 0, 65], None), ([2000, 70], 2000), ([300], 8)],
                         ids=str)
def test_rounded_once(lens, longest, how):
    case(f"output norm of prompts {lens}, max_seqlen {longest}, {how}")
    hk, hv = (1, 2) if max(lens) > 1000 else (2, 6)
    x = lu.inputs(100 + sum(lens), sum(lens) + 40, hk, hv, norm=True, slots=len(lens), **how)
    if how:
        x["w"] = x["w"].float()
    check(x, lens, first=33, max_seqlen=longest)


@pytest.mark.parametrize("delta", [True, False])
def test_chunks_walked_token_by_token(delta):
    """The waves of a head that walk a chunk token by token (one of 16 dims does, for a
    value far above the others) take part in its norm."""
    case(f"output norm with a chunk walked token by token, delta {delta}")
    x = lu.inputs(110, 200, 2, 4, raw=False, delta=delta, norm=True)
    _, _, v = lu.split(x["mixed"], 2, 4)
    v[90, 1, 17] = 2.0 ** 40
    x["g"][91, 1] = -60.0
    x["g"][70, 2] = 30.0  # (all waves of the head)
    check(x, [200], max_seqlen=200)


@pytest.mark.parametrize("longest", [5, 70])
@pytest.mark.parametrize("pad", [64, (1 << 23) + 64])
def test_strided_gates(pad, longest):
    """Rows of z apart, by less and by more than 16 MiB."""
    case(f"output norm, rows of z {pad} values apart, max_seqlen {longest}")
    T, hv = longest, 2
    x = lu.inputs(120, T, 1, hv, norm=True)
    buf = torch.zeros(T, hv * D + pad, dtype=torch.bfloat16, device=DEV)
    z = buf[:, 8:8 + hv * D].unflatten(1, (hv, D))
    z.copy_(x["z"])
    check(x, [T], z=z, max_seqlen=T)


def test_slots_outside_the_pool():
    case("output norm of sequences whose slot is outside the pool")
    for longest in (5, 40, 1500):
        x = lu.inputs(130, longest + 9, 1, 2, norm=True, slots=1)
        gx = lu.on_gpu(x)
        out = torch.full((longest + 9, 2, D), 7.0, device=DEV).bfloat16()
        prompt(gx, ints([4, 0]), ints([2, 2 + longest, longest + 7]), gx["state"], out=out,
               max_seqlen=longest)
        with pytest.raises(_lib.MkvDeviceError, match="state-pool slot"):
            la.check_errors(DEV)
        assert not out[2:2 + longest].any() and out[2 + longest:-2].any()
        assert (out[:2] == 7).all() and (out[-2:] == 7).all()


def test_offsets_that_do_not_hold_together():
    case("output norm, bad offsets in every form")
    x = lu.inputs(131, 1600, 1, 2, norm=True, slots=2)
    gx = lu.on_gpu(x)
    for longest in (5, 40, 1500):
        for cu in ([0, 1601, 1600], [-1, 10, 20], [0, 40, 20]):
            out = torch.full((1600, 2, D), 7.0, device=DEV).bfloat16()
            prompt(gx, ints([0, 1]), ints(cu), gx["state"], out=out, max_seqlen=longest)
            with pytest.raises(_lib.MkvDeviceError, match="inconsistent offsets"):
                la.check_errors(DEV)
            assert (out == 7).all() and torch.equal(gx["state"].cpu(), x["state"])


def test_norm_in_a_captured_graph():
    case("output norm of prompts in a captured graph")
    for lens in ([4, 7], [70, 130], [1500, 60]):
        x = lu.on_gpu(lu.inputs(132, sum(lens), 2, 8, norm=True, slots=2))
        cu, slots = ints([0, lens[0], sum(lens)]), ints([1, 0])
        states = [x["state"].clone() for _ in range(2)]
        run = lambda st: prompt(x, slots, cu, st, max_seqlen=max(lens))  # noqa: E731
        run(states[0].clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(states[0])
        for _ in range(3):
            graph.replay()
            want = run(states[1])
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(states[0], states[1])
    la.check_errors(DEV)
