"""Linear attention, prompt conv and gated norm: what the library refuses, on
the CPU (argument checks come before any use of a pointer), and the oracle's
own closed forms."""
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels import linear_attention as la
from oracle import linear as ref
from tests.test_abi import FAKE, _rc


def decode(**change):
    a = dict(state=FAKE, pool=4, hk=2, hv=8, dim=128, slots=FAKE, batch=3, q=FAKE, qs=512, k=FAKE,
             ks=512, v=FAKE, vs=2048, g=FAKE, gs=32, beta=FAKE, bs=32, bf16=0, a_log=None, dt=None,
             qk=1, scale=0.1, z=None, zs=0, w=None, wb=0, eps=1e-6, out=FAKE, err=FAKE, stream=None)
    a.update(change)
    return _rc("mkv_linear_attn_decode", *a.values())


def prefill(**change):
    a = dict(state=FAKE, pool=4, hk=2, hv=8, dim=128, slots=FAKE, cu=FAKE, batch=3, tokens=5,
             longest=5, q=FAKE, qs=512, k=FAKE, ks=512, v=FAKE, vs=2048, g=FAKE, gs=32, beta=FAKE,
             bs=32, bf16=0, a_log=None, dt=None, qk=1, scale=0.1, z=None, zs=0, w=None, wb=0,
             eps=1e-6, out=FAKE, ws=FAKE, wsb=1 << 40, err=FAKE, stream=None)
    a.update(change)
    return _rc("mkv_linear_attn_prefill", *a.values())


BAD = [
    (dict(state=None), -1, "null pointer"),
    (dict(out=None), -1, "null pointer"),
    (dict(pool=-1), -1, "bad sizes"),
    (dict(hk=0), -1, "bad sizes"),
    (dict(dim=64), -3, "head_dim 64"),
    (dict(hk=3), -3, "8 value heads on 3 key heads"),
    (dict(hv=2048, vs=1 << 20, gs=1 << 14, bs=1 << 14), -3, "at most 1024"),
    (dict(batch=65536), -3, "batch above 65535"),
    (dict(qs=496), -1, "shorter than its row"),
    (dict(gs=16), -1, "shorter than its row"),
    (dict(bs=16), -1, "shorter than its row"),
    (dict(qs=520), -2, "16-byte aligned"),
    (dict(v=FAKE + 2), -2, "16-byte aligned"),
    (dict(g=FAKE + 2), -2, "aligned to their type"),
    (dict(a_log=FAKE), -1, "come together"),
    (dict(z=FAKE, zs=2048), -1, "come together"),
    (dict(z=FAKE, zs=1024, w=FAKE), -1, "shorter than its row"),
]


@pytest.mark.parametrize("change,code,text", BAD)
def test_refused(change, code, text):
    for call in (decode, prefill):
        rc, msg = call(**change)
        assert rc == code and text in msg, msg


def test_prefill_refused():
    assert prefill(cu=None)[0] == -1
    assert prefill(tokens=1 << 31)[0] == -1
    assert prefill(longest=-1)[0] == -1
    assert prefill(vs=(1 << 24) + 16)[0] == -3
    rc, msg = prefill(wsb=8)
    assert rc == -1 and "workspace" in msg
    rc, msg = prefill(ws=FAKE + 8)
    assert rc == -1 and "workspace" in msg
    size = _lib.load().mkv_linear_attn_prefill_workspace_bytes
    assert size(-1, 1, 1, 2, 8, 1) == -1 and size(5, 1, 5, 0, 8, 1) == -1
    assert size(5, 1, 5, 2, 8, 1) > 0


def test_nothing_to_do():
    assert decode(batch=0, state=None)[0] == 0
    assert prefill(batch=0, state=None)[0] == 0
    assert prefill(tokens=0, state=None)[0] == 0
    assert _rc("mkv_gated_rms_norm", None, 256, None, 256, 0, 1, 128, None, 0, 1e-6, None,
               None)[0] == 0
    assert _rc("mkv_gdn_conv_prefill", None, 4, 64, 4, None, None, 0, 0, None, 128, None, 4, None,
               None, None)[0] == 0


def test_conv_prefill_refused():
    def rc(pool=FAKE, channels=64, width=4, cu=FAKE, tokens=9, x=FAKE, xs=128, kernel=4, out=FAKE):
        return _rc("mkv_gdn_conv_prefill", pool, 4, channels, width, FAKE, cu, 2, tokens, x, xs,
                   FAKE, kernel, out, FAKE, None)
    assert rc(pool=None)[0] == -1 and rc(cu=None)[0] == -1 and rc(tokens=-1)[0] == -1
    assert rc(width=5)[0] == -3 and rc(kernel=3)[0] == -3 and rc(channels=60)[0] == -3
    assert rc(xs=112)[0] == -1 and rc(xs=136)[0] == -2 and rc(x=FAKE + 8)[0] == -2


def test_gated_norm_refused():
    def rc(x=FAKE, xs=256, tokens=3, heads=1, dim=128, w=FAKE, wb=1):
        return _rc("mkv_gated_rms_norm", x, xs, FAKE, 256, tokens, heads, dim, w, wb, 1e-6, FAKE,
                   None)
    assert rc(x=None)[0] == -1 and rc(tokens=-1)[0] == -1 and rc(heads=0)[0] == -1
    assert rc(dim=100)[0] == -3 and rc(dim=4104)[0] == -3
    assert rc(xs=128)[0] == -1 and rc(xs=264)[0] == -2 and rc(w=FAKE + 1)[0] == -2
    assert rc(tokens=(1 << 32) + 1)[0] == -3


def test_tensors_off_the_gpu_raise():
    x = torch.zeros(2, 1, 128, dtype=torch.bfloat16)
    g = torch.zeros(2, 1)
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        la.linear_attn_decode(x, x, x, g, g, torch.zeros(4, 1, 128, 128), torch.arange(2))
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        la.gated_rms_norm(x, x, torch.ones(128))


def test_oracle_closed_forms():
    """Without decay and delta rule S is the sum of u k^T; with the delta rule
    and beta = 1 a unit key reads its value back at once; a decay of e^-inf
    forgets."""
    g = torch.Generator().manual_seed(5)
    q = torch.randn(6, 2, 8, generator=g)
    k = torch.randn(6, 2, 8, generator=g)
    v = torch.randn(6, 4, 8, generator=g)
    none = torch.zeros(6, 4)
    o, s, _ = ref.scan(q, k, v, none, None, torch.zeros(4, 8, 8), 1.0)
    kk = k.double().repeat_interleave(2, 1)
    assert torch.allclose(s, torch.einsum("thv,thk->hvk", v.double(), kk))
    assert torch.allclose(o[-1], (s * q[-1].double().repeat_interleave(2, 0)[:, None, :]).sum(-1))
    k = k / k.norm(dim=-1, keepdim=True)
    o, s, _ = ref.scan(k, k, v, none, torch.ones(6, 4), torch.randn(4, 8, 8, generator=g), 1.0)
    assert torch.allclose(o, v.double(), atol=1e-5)
    o, s, _ = ref.scan(q, k, v, torch.full((6, 4), -float("inf")), None,
                       torch.randn(4, 8, 8, generator=g), 1.0)
    assert torch.allclose(s, v[-1].double()[:, :, None] * k[-1].double().repeat_interleave(
        2, 0)[:, None, :])
    one = ref.gated_norm(torch.full((1, 8), 3.0), torch.zeros(1, 8), torch.ones(8), 0.0)
    assert (one == 0).all()
    g, beta = ref.gates(torch.zeros(1, 1), torch.zeros(1, 1), torch.zeros(1), torch.zeros(1))
    assert torch.allclose(g, torch.tensor(-0.6931471805599453).double()) and beta == 0.5


def test_more_sequences_and_rows_than_a_call_takes():
    assert prefill(batch=4096, cu=None)[0] == -1  # (4096 are taken: the next check speaks)
    rc, msg = prefill(batch=4097)
    assert rc == -3 and "more than 4096 sequences" in msg
    rc, msg = prefill(tokens=(1 << 27) + 1)
    assert rc == -3 and "too many rows" in msg
    rc, msg = _rc("mkv_gdn_conv_prefill", FAKE, 4, 64, 4, FAKE, FAKE, 4097, 9, FAKE, 128, FAKE, 4,
                  FAKE, FAKE, None)
    assert rc == -3 and "more than 4096 sequences" in msg
    rc, msg = _rc("mkv_gdn_conv_prefill", FAKE, 4, 64, 4, FAKE, FAKE, 2, (1 << 27) + 1, FAKE, 128,
                  FAKE, 4, FAKE, FAKE, None)
    assert rc == -3 and "too many rows" in msg
    rc, msg = _rc("mkv_gated_rms_norm", FAKE, 256, FAKE, 256, (1 << 29) + 1, 2, 64, FAKE, 0, 1e-6,
                  FAKE, None)
    assert rc == -3 and "too many rows" in msg


def test_workspace_of_many_heads_on_one_key_head():
    """Value heads of one key head run in turn where their images would take more than
    2 GiB; what is joined of segments comes on top."""
    size = _lib.load().mkv_linear_attn_prefill_workspace_bytes
    for tokens in (300000, 1000000):
        for delta in (0, 1):
            assert 1 << 30 < size(tokens, 2, tokens, 1, 64, delta) < 3 << 30
    assert size(32768, 8, 4096, 2, 8, 1) < 1 << 29


def test_rows_of_one_head_that_a_launch_does_not_take():
    """2^29 rows of one head are 2^23 chunks of 512 threads: as many as a grid dimension
    has; a little less passes (the next check speaks)."""
    one = dict(hk=1, hv=1, qs=256, ks=256, vs=256, gs=4, bs=4, longest=0, wsb=8)
    rc, msg = prefill(tokens=1 << 29, **one)
    assert rc == -3 and "too many rows" in msg
    rc, msg = prefill(tokens=(1 << 29) - 512, batch=7, **one)
    assert rc == -1 and "workspace" in msg
