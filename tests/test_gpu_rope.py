"""The norm of query and key heads with the rotation, by itself and with the paged append,
against the float64 oracle.

Tolerance: half a step of the output's type (bf16 2^-8, fp16 2^-11 of the value, 2^-25 below
fp16's normal range), and of |y_i c| + |y_j s| what fp32 is off: 2^-19 covers the sum of 256
squares (13 roundings of 2^-24), the root and its product with the weight (5), sine and cosine
(2^-22 with the angle's rounding) and the last two products and sum (3)."""
import numpy as np
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels import attention as A
from muserve_amd.kernels.rope import qk_norm_rope
from muserve_amd.kv_cache import PagedKVCache
from oracle import attention as att
from oracle import fp4
from oracle import rope as ref
from tests.gpu_util import DEV, case

pytestmark = pytest.mark.gpu
POOLS = [torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2]


def close(got, x, positions, freq, weight, **how):
    want, size = ref.norm_rope(x.double().cpu().numpy(), positions.cpu().numpy(),
                               freq.double().cpu().numpy(),
                               None if weight is None else weight.double().cpu().numpy(), **how)
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -11
    low = 0.0 if got.dtype == torch.bfloat16 else 2.0 ** -25
    err = np.abs(got.double().cpu().numpy() - want)
    tol = half * np.abs(want) + low + 2.0 ** -19 * size
    assert (err <= tol).all(), f"{(err > tol).sum()} of {err.size} off, worst {(err / tol).max()}"


def inputs(seed, tokens, hq, hk, dim, dtype, rot, far=32768, gate=False, weights=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    wide = 2 * dim if gate else dim
    x = (3 * torch.randn(tokens, hq * wide + 2 * hk * dim, generator=g)).to(dtype).to(DEV)
    q = x[:, :hq * wide].unflatten(1, (hq, wide))[..., :dim]
    k = x[:, hq * wide:hq * wide + hk * dim].unflatten(1, (hk, dim))
    v = x[:, hq * wide + hk * dim:].unflatten(1, (hk, dim))
    pos = torch.randint(0, far, (tokens,), generator=g).to(DEV)
    freq = (1e6 ** (-torch.arange(0, rot, 2).double() / rot)).float().to(DEV)
    qw, kw = ((1 + 0.2 * torch.randn(dim, generator=g)).to(weights).to(DEV) for _ in range(2))
    return q, k, v, pos, freq, qw, kw


@pytest.mark.parametrize("dim,rot", [(256, 64), (256, 256), (256, 48), (128, 128), (128, 32),
                                     (64, 64), (64, 16), (64, 48)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_dims_and_styles(dim, rot, interleaved, dtype):
    case(f"norm + rotation: head dim {dim}, {rot} turned, interleaved {interleaved}, {dtype}")
    q, k, _, pos, freq, qw, kw = inputs(dim + rot, 37, 4, 1, dim, dtype, rot, gate=True)
    qo, ko = qk_norm_rope(q, k, pos, freq, qw, kw, interleaved=interleaved)
    torch.cuda.synchronize()
    close(qo, q, pos, freq, qw, interleaved=interleaved)
    close(ko, k, pos, freq, kw, interleaved=interleaved)


@pytest.mark.parametrize("tokens,hq,hk", [(1, 4, 1), (2, 1, 1), (7, 32, 2), (300, 3, 3), (1, 1, 0),
                                          (5, 0, 2), (4097, 4, 1), (1000, 9, 3)])
def test_tokens_and_heads(tokens, hq, hk):
    case(f"norm + rotation: {tokens} tokens, {hq} and {hk} heads")
    q, k, _, pos, freq, qw, kw = inputs(tokens, tokens, hq, hk, 256, torch.bfloat16, 64)
    qo, ko = qk_norm_rope(q, k, pos, freq, qw, kw, zero_centered=True)
    torch.cuda.synchronize()
    assert qo.shape == q.shape and ko.shape == k.shape and ko.is_contiguous()
    close(qo, q, pos, freq, qw, zero_centered=True)
    close(ko, k, pos, freq, kw, zero_centered=True)


@pytest.mark.parametrize("weights", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("which", ["both", "q", "k", "none"])
def test_weights(weights, which):
    case(f"norm + rotation: weights {weights}, {which}")
    q, k, _, pos, freq, qw, kw = inputs(3, 21, 2, 2, 128, torch.bfloat16, 64, weights=weights)
    qw = qw if which in ("both", "q") else None
    kw = kw if which in ("both", "k") else None
    qo, ko = qk_norm_rope(q, k, pos, freq, qw, kw, 1e-5, rope_scale=1.25)
    torch.cuda.synchronize()
    close(qo, q, pos, freq, qw, eps=1e-5, rope_scale=1.25)
    close(ko, k, pos, freq, kw, eps=1e-5, rope_scale=1.25)


def test_far_positions_and_frequency_types():
    case("norm + rotation: far and negative positions, fp64 frequencies")
    q, k, _, _, freq, qw, kw = inputs(4, 8, 2, 1, 256, torch.float16, 64)
    pos = torch.tensor([0, 1, 262143, 1048575, 16777217, 2 ** 31 - 1, -5, -262144], device=DEV)
    for f in (freq, freq.double() * (1 + 1e-9)):
        for p in (pos, pos.int()):
            qo, ko = qk_norm_rope(q, k, p, f, qw, kw)
            torch.cuda.synchronize()
            close(qo, q, p, f, qw)
            close(ko, k, p, f, kw)


def test_rows_of_zeros_large_and_small_values():
    case("norm + rotation: zeros, large and small values")
    q, k, _, pos, freq, qw, kw = inputs(5, 6, 1, 1, 256, torch.bfloat16, 64)
    q = q.contiguous()
    q[0] = 0
    q[1] *= 1e15
    q[2] *= 1e-15
    q[3, 0, 1:] = 0
    qo, ko = qk_norm_rope(q, k, pos, freq, qw, kw)
    torch.cuda.synchronize()
    close(qo, q, pos, freq, qw)
    q[4, 0, 200] = float("nan")
    qo, _ = qk_norm_rope(q, k, pos, freq, qw, kw)
    assert qo[4].isnan().all() and not qo[[0, 1, 2, 3, 5]].isnan().any()


def test_in_place_and_given_outputs():
    case("norm + rotation: in place, and into given tensors")
    q, k, _, pos, freq, qw, kw = inputs(6, 33, 4, 2, 256, torch.bfloat16, 64)
    want = qk_norm_rope(q, k, pos, freq, qw, kw)
    a, b = q.contiguous().clone(), k.contiguous().clone()
    got = qk_norm_rope(a, b, pos, freq, qw, kw, out=(a, b))
    torch.cuda.synchronize()
    assert got[0] is a and torch.equal(a, want[0]) and torch.equal(b, want[1])
    out = (torch.empty_like(want[0]), torch.empty_like(want[1]))
    qk_norm_rope(q, k, pos, freq, qw, kw, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("dtype", POOLS)
@pytest.mark.parametrize("heads", [(4, 1), (8, 2), (9, 3)])
@pytest.mark.parametrize("tokens", [1, 45, 700])
def test_append_rope_is_the_norm_and_the_append(dtype, heads, tokens):
    """Bit for bit what qk_norm_rope and append leave, skipped tokens included."""
    case(f"append_rope: pool {dtype}, {heads} heads, {tokens} tokens")
    hq, hk = heads
    value = torch.float16 if dtype == torch.float16 else torch.bfloat16
    q, k, v, pos, freq, qw, kw = inputs(tokens, tokens, hq, hk, 256, value, 64, gate=True)
    pages = -(-tokens // 16) + 4
    g = torch.Generator().manual_seed(tokens)
    slots = torch.randperm(pages * 16, generator=g)[:tokens]
    if tokens > 1:
        slots[3] = -1
    a, b = (PagedKVCache(pages, num_layers=2, kv_heads=hk, dtype=dtype, device=DEV, verbose=False)
            for _ in range(2))
    got = a.append_rope(slots.to(DEV), q, k, v, 1, pos, freq, qw, kw, zero_centered=True)
    want, turned = qk_norm_rope(q, k, pos, freq, qw, kw, zero_centered=True)
    b.append(slots.to(DEV), turned, v.contiguous(), layer=1)
    a.check_errors()
    b.check_errors()
    assert torch.equal(got, want)
    assert torch.equal(a.cache.view(torch.uint8), b.cache.view(torch.uint8))
    if a.scales is not None:
        assert torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("dim", [64, 128])
def test_append_rope_of_other_dims(dim):
    case(f"append_rope: head dim {dim}")
    q, k, v, pos, freq, qw, kw = inputs(dim, 50, 6, 2, dim, torch.float16, 32)
    cache = PagedKVCache(8, num_layers=1, kv_heads=2, head_dim=dim, dtype=torch.float16, device=DEV,
                         verbose=False)
    slots = torch.arange(30, 80, device=DEV)
    out = torch.empty(50, 6, dim, dtype=torch.float16, device=DEV)
    assert cache.append_rope(slots, q, k, v, 0, pos.int(), freq, qw, kw, interleaved=True,
                             out=out) is out
    cache.check_errors()
    close(out, q, pos, freq, qw, interleaved=True)
    flat = cache.cache[0].view(2, 128, 2, dim)
    close(flat[0, 30:80], k, pos, freq, kw, interleaved=True)
    assert torch.equal(flat[1, 30:80], v) and not flat[:, :30].any() and not flat[:, 80:].any()


def test_append_rope_flags_bad_slots():
    case("append_rope: slots outside the pool, and twice the same")
    q, k, v, pos, freq, qw, kw = inputs(8, 3, 4, 1, 256, torch.bfloat16, 64)
    cache = PagedKVCache(2, num_layers=1, kv_heads=1, dtype=torch.bfloat16, device=DEV,
                         verbose=False)
    for bad in (32, -2, 1 << 40):
        out = cache.append_rope(torch.tensor([4, bad, 9], device=DEV), q, k, v, 0, pos, freq, qw, kw)
        with pytest.raises(_lib.MkvDeviceError, match="slot_mapping"):
            cache.check_errors()
        close(out, q, pos, freq, qw)
    written = torch.zeros(32, dtype=torch.bool)
    written[[4, 9]] = True
    assert torch.equal(cache.cache[0, 1].view(32, -1).any(-1).cpu(), written)
    cache.check_unique = True
    cache.append_rope(torch.tensor([5, 5, 9], device=DEV), q, k, v, 0, pos, freq, qw, kw)
    with pytest.raises(_lib.MkvDeviceError, match="more than once"):
        cache.check_errors()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float4_e2m1fn_x2])
def test_a_decode_layer(dtype):
    """append_rope, then the decode attention over what it left, step after step, captured."""
    case(f"a decode layer over {dtype}")
    B, hq, hk, steps = 5, 4, 1, 20
    cache = PagedKVCache(24, num_layers=1, kv_heads=hk, dtype=dtype, device=DEV, verbose=False)
    order = torch.randperm(24, generator=torch.Generator().manual_seed(1))[:20].view(B, 4)
    table = order.int().to(DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    slots = torch.zeros(B, dtype=torch.int64, device=DEV)
    pos = torch.zeros(B, dtype=torch.int64, device=DEV)
    q, k, v, _, freq, qw, kw = (x.contiguous() for x in inputs(9, B, hq, hk, 256, torch.bfloat16, 64))
    attend = A.attn_decode_fp4 if dtype == torch.float4_e2m1fn_x2 else A.attn_decode

    def layer():
        turned = cache.append_rope(slots, q, k, v, 0, pos, freq, qw, kw)
        return turned, attend(turned[:, None], *cache.get_kv_by_layer(0), lens, table)

    slots.fill_(-1)
    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, out = layer()
    starts = torch.tensor([0, 3, 15, 16, 31])
    cache.append(torch.cat([order[b, p // 16] * 16 + p % 16 for b in range(B)
                            for p in [torch.arange(starts[b])]]).to(DEV),
                 *(torch.randn(int(starts.sum()), hk, 256).bfloat16().to(DEV) for _ in range(2)),
                 layer=0)
    for step in range(steps):
        at = starts + step
        pos.copy_(at)
        lens.copy_(at + 1)
        slots.copy_(order[torch.arange(B), at // 16] * 16 + at % 16)
        q.copy_(torch.randn(B, hq, 256))
        k.copy_(torch.randn(B, hk, 256))
        v.copy_(torch.randn(B, hk, 256))
        graph.replay()
        torch.cuda.synchronize()
        cache.check_errors()
        A.check_errors(DEV)
        close(turned, q, pos, freq, qw)
        kc, vc = ((fp4.values(x.cpu().numpy()) if dtype != torch.bfloat16 else x.double().cpu().numpy())
                  for x in cache.get_kv_by_layer(0))
        want, mass, smax = att.decode_attention(turned.double().cpu().numpy(), kc, vc,
                                                (at + 1).numpy(), table.cpu().numpy(), 256 ** -0.5,
                                                stats=True)
        tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -14 + 2.0 ** -16 * (1 + smax[..., None])) * mass
        assert (np.abs(out[:, 0].double().cpu().numpy() - want) <= tol).all()


def test_a_prefill_chunk_over_a_4_bit_pool():
    """Two chunks by append_rope, their window read back, prefill attention over it."""
    case("a prefill chunk over a 4-bit pool")
    lens, chunk, hq, hk = [70, 45], [30, 45], 4, 1
    cache = PagedKVCache(16, num_layers=1, kv_heads=hk, dtype=torch.float4_e2m1fn_x2, device=DEV,
                         verbose=False)
    order = torch.randperm(16, generator=torch.Generator().manual_seed(2))[:10].view(2, 5)
    freq = (1e6 ** (-torch.arange(0, 64, 2).double() / 64)).float().to(DEV)

    def at(b, start, n):
        p = torch.arange(start, start + n)
        return order[b, p // 16] * 16 + p % 16, p

    for spans in ([(0, 0, 40)], [(0, 40, 30), (1, 0, 45)]):
        both = [at(*s) for s in spans]
        slots, pos = (torch.cat(x).to(DEV) for x in zip(*both))
        q, k, v, _, _, qw, kw = inputs(len(spans), len(pos), hq, hk, 256, torch.bfloat16, 64)
        turned = cache.append_rope(slots, q, k, v, 0, pos, freq, qw, kw)
    cu_k = torch.tensor([0, 70, 115], device=DEV)
    kw_, vw = cache.gather(0, order.int().to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                           out_len=70, cu_out=cu_k)
    out = A.attn_prefill(turned, kw_, vw, torch.tensor([0, 30, 75], device=DEV, dtype=torch.int32),
                         cu_k.int(), 45, 70)
    torch.cuda.synchronize()
    cache.check_errors()
    kc, vc = (fp4.values(x.cpu().numpy()) for x in cache.get_kv_by_layer(0))
    want, mass = att.prefill_attention(turned.double().cpu().numpy(), kc, vc, [0, 30, 75], 1 / 16,
                                       lens_k=lens, page_table=order.numpy(), stats=True)
    tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -8 * mass
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


def test_refusals():
    case("norm + rotation: refused arguments")
    q, k, v, pos, freq, qw, kw = inputs(10, 6, 4, 1, 256, torch.bfloat16, 64)

    def refused(error, **change):
        args = dict(q=q, k=k, positions=pos, inv_freq=freq, q_weight=qw, k_weight=kw)
        args.update(change)
        with pytest.raises(error):
            qk_norm_rope(**args)

    refused(TypeError, q=q.float(), k=k.float())
    refused(TypeError, k=k.half())
    refused(ValueError, q=q[..., :96], k=k[..., :96])
    refused(ValueError, k=k[:5])
    refused(ValueError, q=q.transpose(1, 2).contiguous().transpose(1, 2))
    refused(ValueError, positions=pos[:5])
    refused(ValueError, positions=pos.float())
    refused(ValueError, inv_freq=freq[:5])
    refused(ValueError, inv_freq=torch.ones(136, device=DEV))
    refused(ValueError, inv_freq=freq.half())
    refused(ValueError, q_weight=qw[:128])
    refused(TypeError, q_weight=qw.float())
    refused(RuntimeError, q=q.cpu())
    # rows that other workgroups still read
    a = q.contiguous()
    refused(ValueError, q=a, out=(a.flip(0)[:5], torch.empty_like(k)))
    both = torch.empty(7, 4, 256, dtype=torch.bfloat16, device=DEV)
    refused(ValueError, q=both[:6], out=(both[1:], k.contiguous()))
    refused(ValueError, q=a, k=a[:, :1], out=(a, torch.empty_like(k.contiguous())))
    cache = PagedKVCache(2, num_layers=1, kv_heads=1, dtype=torch.float16, device=DEV, verbose=False)
    slots = torch.arange(6, device=DEV)
    with pytest.raises(TypeError):
        cache.append_rope(slots, q, k, v, 0, pos, freq, qw, kw)
    cache = PagedKVCache(2, num_layers=1, kv_heads=1, dtype=torch.bfloat16, device=DEV, verbose=False)
    for bad in (dict(layer=1), dict(layer=-2)):
        with pytest.raises(IndexError):
            cache.append_rope(slots, q, k, v, bad["layer"], pos, freq, qw, kw)
    with pytest.raises(ValueError):
        cache.append_rope(slots[:5], q, k, v, 0, pos, freq, qw, kw)
    with pytest.raises(ValueError):
        cache.append_rope(slots, q, torch.cat([k, k], 1), v, 0, pos, freq, qw, kw)
    with pytest.raises(ValueError):
        cache.append_rope(slots, q, k, v[:, :, :128], 0, pos, freq, qw, kw)
    cache.check_errors()
    qo, ko = qk_norm_rope(q[:0], k[:0], pos[:0], freq, qw, kw)
    assert qo.shape == (0, 4, 256) and ko.shape == (0, 1, 256)
