"""append_rope into every kind of pool, in each style, head size and rotary dim that a call may
choose: bit for bit what qk_norm_rope and append leave."""
import pytest
import torch

from muserve_amd.kernels.rope import qk_norm_rope
from muserve_amd.kv_cache import PagedKVCache
from tests.gpu_util import DEV, case

pytestmark = pytest.mark.gpu
POOLS = [torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2]
CASES = [(pool, dim, rot, pairs) for pool in POOLS for dim in (64, 128, 256)
         for rot in (16, 48, dim) for pairs in (False, True)
         if dim == 256 or pool in (torch.bfloat16, torch.float16)]


@pytest.mark.parametrize("pool,dim,rot,pairs", CASES)
@pytest.mark.parametrize("tokens,hq,hk,weights", [(1, 4, 1, torch.bfloat16), (37, 6, 2, torch.float32),
                                                  (601, 3, 3, None)])
def test_append_rope_is_the_norm_and_the_append(pool, dim, rot, pairs, tokens, hq, hk, weights):
    case(f"append_rope: {pool}, heads of {dim}, {rot} turned, pairs {pairs}, {tokens} tokens, "
         f"{hq} and {hk} heads, weights {weights}")
    g = torch.Generator().manual_seed(dim + rot + tokens)
    value = torch.float16 if pool == torch.float16 else torch.bfloat16
    x = (3 * torch.randn(tokens, (hq + 2 * hk) * dim, generator=g)).to(value).to(DEV)
    q, k, v = (y.unflatten(1, (-1, dim)) for y in x.split([hq * dim, hk * dim, hk * dim], 1))
    qw = kw = None
    if weights is not None:
        qw, kw = ((0.2 * torch.randn(dim, generator=g)).to(weights).to(DEV) for _ in range(2))
    freq = (1e6 ** (-torch.arange(0, rot, 2).double() / rot)).to(DEV)
    pos = torch.randint(0, 1 << 18, (tokens,), generator=g).to(DEV)
    pages = -(-tokens // 16) + 3
    slots = torch.randperm(pages * 16, generator=g)[:tokens]
    if tokens > 1:
        slots[torch.randperm(tokens, generator=g)[:3]] = -1
    how = dict(rope_scale=1.25, zero_centered=weights is not None, interleaved=pairs)
    a, b = (PagedKVCache(pages, num_layers=2, kv_heads=hk, head_dim=dim, dtype=pool, device=DEV,
                         verbose=False) for _ in range(2))
    for cache in (a, b):
        cache.cache.view(torch.uint8).fill_(0x2A)
    got = a.append_rope(slots.to(DEV), q, k, v, 1, pos, freq, qw, kw, 1e-5, **how)
    want, turned = qk_norm_rope(q, k, pos, freq, qw, kw, 1e-5, **how)
    b.append(slots.to(DEV), turned, v.contiguous(), layer=1)
    a.check_errors()
    b.check_errors()
    assert torch.equal(got, want) and not got.isnan().any()
    assert torch.equal(a.cache.view(torch.uint8), b.cache.view(torch.uint8))
    if a.scales is not None:
        assert torch.equal(a.scales, b.scales)
