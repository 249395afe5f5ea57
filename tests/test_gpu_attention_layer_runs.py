"""An attention layer's operators over a 4-bit pool as a serving loop uses them: the scheduler's
plan drives the rotation with its append, the decode attention and the prefill chunks' windows;
shared prompt pages; the prefix cache's host tier; outputs in place.

The attention's tolerance is tests/test_gpu_attention_fp4.py's, the prefill attention's is
tests/test_gpu_prefill.py's for bf16 probabilities (2^-8 of the attended mass)."""
import numpy as np
import pytest
import torch

from muserve_amd.kernels import attention as A
from muserve_amd.kernels.rope import qk_norm_rope
from muserve_amd.kv_cache import PagedKVCache
from muserve_amd.model.prefix_cache import PrefixCache
from muserve_amd.scheduler import ContinuousBatchScheduler, InferenceRequest
from oracle import attention as att
from oracle import fp4
from tests.gpu_util import DEV, case

pytestmark = pytest.mark.gpu
FP4 = torch.float4_e2m1fn_x2
FREQ = 1e6 ** (-torch.arange(0, 64, 2).double() / 64)


def make_pool(pages, layers=1, heads=1):
    return PagedKVCache(pages, num_layers=layers, kv_heads=heads, dtype=FP4, device=DEV,
                        verbose=False)


def values(cache, layer=0):
    return (fp4.values(x.cpu().numpy()) for x in cache.get_kv_by_layer(layer))


def decode_close(got, q, cache, lens, table, layer=0):
    k, v = values(cache, layer)
    want, mass, smax = att.decode_attention(q.double().cpu().numpy(), k, v, lens, table, 1 / 16,
                                            stats=True)
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -14 + 2.0 ** -16 * (1 + smax[..., None])) * mass
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("hq,hk", [(4, 1), (8, 2)])
def test_a_scheduler_drives_the_layer(hq, hk):
    case(f"scheduler plan -> append_rope -> decode and prefill attention, {hq} heads on {hk}")
    rng = np.random.default_rng(4)
    g = torch.Generator(device=DEV).manual_seed(4)
    cache = make_pool(256, heads=hk)
    cache._free_pages = rng.permutation(256).tolist()
    s = ContinuousBatchScheduler(max_batch_size=6, max_seq_len=512, kv_cache=cache,
                                 chunked_prefill_size=96)
    for i in range(10):
        s.add_request(InferenceRequest(request_id=i, input_ids=list(range(int(rng.integers(1, 200)))),
                                       max_new_tokens=int(rng.integers(1, 12))))
    freq = FREQ.float().to(DEV)
    qw, kw = (0.1 * torch.randn(256, device=DEV, generator=g) for _ in range(2))
    decoded = prefilled = 0
    while True:
        plan = s.plan_step()
        if plan is None:
            break
        T, nd = plan.num_tokens, plan.num_decode
        x = torch.randn(T, (2 * hq + 2 * hk) * 256, device=DEV, generator=g).bfloat16()
        q = x[:, :2 * hq * 256].unflatten(1, (hq, 512))[..., :256]
        k, v = (y.unflatten(1, (hk, 256)) for y in x[:, 2 * hq * 256:].chunk(2, 1))
        turned = cache.append_rope(plan.slot_mapping, q, k, v, 0, plan.positions, freq, qw, kw,
                                   zero_centered=True)
        lens, table = plan.seq_lens.cpu().numpy(), plan.block_tables.cpu().numpy()
        if nd and decoded < 8:
            out = A.attn_decode_fp4(turned[:nd, None], *cache.get_kv_by_layer(0),
                                    plan.seq_lens[:nd], plan.block_tables[:nd])
            decode_close(out[:, 0], turned[:nd], cache, lens[:nd], table[:nd])
            decoded += 1
        n = len(lens) - nd
        if n and prefilled < 6 and hq == 4 * hk:
            cu = torch.tensor([0, *np.cumsum(lens[nd:])], device=DEV)
            kw_, vw = cache.gather(0, plan.block_tables[nd:], plan.seq_lens[nd:],
                                   out_len=int(lens[nd:].max()), cu_out=cu)
            cu_q = (plan.cu_seqlens[nd:] - nd).int()
            out = A.attn_prefill(turned[nd:], kw_, vw, cu_q, cu.int(), T - nd, int(lens[nd:].max()))
            kc, vc = values(cache)
            want, mass = att.prefill_attention(turned[nd:].double().cpu().numpy(), kc, vc,
                                               cu_q.cpu().numpy(), 1 / 16, lens_k=lens[nd:],
                                               page_table=table[nd:], stats=True)
            err = np.abs(out.double().cpu().numpy() - want)
            assert (err <= 2.0 ** -8 * np.abs(want) + 2.0 ** -8 * mass).all()
            prefilled += 1
        s.complete_step(plan, rng.integers(4, 64, len(plan.entries)).tolist())
    cache.check_errors()
    A.check_errors(DEV)
    assert decoded >= 5 and prefilled >= 4


def test_pages_shared_and_copied():
    """Two sequences on one prompt's pages, the second continuing on a copy of the last one."""
    case("4-bit pool: shared prompt pages and a copied one")
    cache = make_pool(12, layers=2)
    g = torch.Generator().manual_seed(5)
    table = torch.tensor([[7, 2, 9], [7, 2, 4]], dtype=torch.int32)
    x = torch.randn(2, 2, 40, 1, 256, generator=g).bfloat16().to(DEV)
    pos = torch.arange(40)
    slots = table[0].long()[pos // 16] * 16 + pos % 16
    cache.append(slots.to(DEV), x[:, 0], x[:, 1])
    cache.copy_pages([9], [4])
    more = torch.randn(2, 1, 256, generator=g).bfloat16().to(DEV)
    cache.append(torch.tensor([9 * 16 + 8, 4 * 16 + 8], device=DEV), more, -more, layer=1)
    q = torch.randn(2, 1, 4, 256, generator=g).bfloat16().to(DEV)
    out = A.attn_decode_fp4(q, *cache.get_kv_by_layer(1),
                            torch.tensor([41, 41], dtype=torch.int32, device=DEV), table.to(DEV),
                            shared_pages=8)
    cache.check_errors()
    A.check_errors(DEV)
    decode_close(out[:, 0], q[:, 0], cache, np.array([41, 41]), table.numpy(), layer=1)


def test_the_prefix_cache_keeps_4_bit_pages():
    case("PrefixCache with a prefix's pages of a 4-bit pool")
    cache = make_pool(64, layers=3, heads=2)
    x = torch.randn(2, 3, 1024, 2, 256, generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    cache.append(torch.arange(1024, device=DEV), x[0], x[1])
    ids = torch.arange(90, dtype=torch.int64)
    pages = cache.alloc_pages(5)
    before = cache.cache[:, :, pages].clone()
    pc = PrefixCache(max_entries=2, host_bytes=8 << 20)
    pc.store(ids.to(DEV), 70, torch.ones(70, 8, device=DEV), [None], kv=(cache, pages))
    cache.free_pages(pages)
    cache.cache.zero_()
    hit = pc.lookup_kv(ids, DEV, cache)
    torch.cuda.synchronize()
    pc.sync()
    assert hit[0] == 70 and torch.equal(cache.cache[:, :, hit[3]], before)


def test_outputs_in_place_and_overlapping():
    case("decode attention and append_rope: in place, and outputs that overlap")
    g = torch.Generator().manual_seed(7)
    cache = make_pool(8)
    x = torch.randn(2, 128, 1, 256, generator=g).bfloat16().to(DEV)
    cache.append(torch.arange(128, device=DEV), x[0], x[1], layer=0)
    k, v = cache.get_kv_by_layer(0)
    table = torch.arange(8, dtype=torch.int32).view(2, 4).to(DEV)
    for lens in ([60, 33], [1, 64]):
        ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
        q = torch.randn(2, 1, 4, 256, generator=g).bfloat16().to(DEV)
        want = A.attn_decode_fp4(q, k, v, ln, table)
        assert A.attn_decode_fp4(q, k, v, ln, table, out=q) is q
        torch.cuda.synchronize()
        assert torch.equal(q, want)
    both = torch.empty(3, 1, 4, 256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        A.attn_decode_fp4(both[:2], k, v, ln, table, out=both[1:])
    pool = PagedKVCache(8, num_layers=1, kv_heads=1, dtype=torch.bfloat16, device=DEV, verbose=False)
    q = torch.randn(5, 4, 256, generator=g).bfloat16().to(DEV)
    kv = torch.randn(2, 5, 1, 256, generator=g).bfloat16().to(DEV)
    freq, pos = FREQ.float().to(DEV), torch.arange(5, device=DEV)
    want = qk_norm_rope(q, kv[0], pos, freq)[0]
    slots = torch.arange(5, device=DEV)
    assert pool.append_rope(slots, q, kv[0], kv[1], 0, pos, freq, out=q) is q
    torch.cuda.synchronize()
    assert torch.equal(q, want)
    inside = pool.cache.view(-1)[:q.numel()].view(q.shape)
    with pytest.raises(ValueError, match="overlaps"):
        pool.append_rope(slots, q, kv[0], kv[1], 0, pos, freq, out=inside)


def test_unaligned_rows_are_refused():
    case("norm + rotation: rows at odd addresses")
    freq, pos = FREQ.float().to(DEV), torch.arange(2, device=DEV)
    flat = torch.zeros(2 * 256 + 4, dtype=torch.bfloat16, device=DEV)
    odd = flat[4:].view(2, 1, 256)
    even = torch.zeros(2, 1, 256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="misaligned"):
        qk_norm_rope(odd, even, pos, freq)
    with pytest.raises(RuntimeError, match="misaligned"):
        qk_norm_rope(even, even.clone(), pos, freq, out=(odd, torch.empty_like(even)))
    torch.cuda.synchronize()


def random_rows(rng, *shape):
    rows = rng.integers(0, 256, (*shape, fp4.ROW), dtype=np.uint8)
    rows[..., 128:] = rng.integers(122, 130, (*shape, 8))
    return rows


@pytest.mark.parametrize("lens,hq,hkv", [
    ([40, 3], 520, 520),                     # more KV heads than the grid has places for
    ([30000, 17000], 4, 2), ([20001], 6, 3), ([9000, 0, 8191], 10, 2),
    ([8160], 4, 1), ([8192], 4, 1),          # around the joining kernel's width
    ([9] * 2047 + [70], 2, 2),               # the most pairs of a call
    ([2000, 1, 700] * 60, 8, 1)])
def test_shapes_of_heads(lens, hq, hkv):
    case(f"4-bit decode attention: {len(lens)} sequences, longest {max(lens)}, {hq} heads on {hkv}")
    rng = np.random.default_rng(hq + len(lens))
    pages = [-(-n // 16) for n in lens]
    P = sum(pages) + 2
    perm = rng.permutation(P)
    table = np.zeros((len(lens), max(pages)), dtype=np.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    k, v = random_rows(rng, P, 16, hkv), random_rows(rng, P, 16, hkv)
    q = (0.2 * torch.randn(len(lens), 1, hq, 256,
                           generator=torch.Generator().manual_seed(hq))).bfloat16()
    out = A.attn_decode_fp4(q.to(DEV), *(torch.from_numpy(x).to(DEV) for x in (k, v)),
                            torch.tensor(lens, dtype=torch.int32, device=DEV),
                            torch.from_numpy(table).to(DEV))
    A.check_errors(DEV)
    want, mass, smax = att.decode_attention(q[:, 0].double().numpy(), fp4.values(k), fp4.values(v),
                                            np.asarray(lens), table, 1 / 16, stats=True)
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -14 + 2.0 ** -16 * (1 + smax[..., None])) * mass
    assert (np.abs(out[:, 0].double().cpu().numpy() - want) <= tol).all()


def test_rows_behind_4_gib():
    """Queries whose rows are 3 GiB apart, pages behind 4 GiB of a plane."""
    case("append_rope: rows and pages behind 4 GiB")
    g = torch.Generator(device=DEV).manual_seed(8)
    step = 3 << 29
    flat = torch.empty(2 * step + 512, dtype=torch.bfloat16, device=DEV)
    q = flat.as_strided((3, 2, 256), (step, 256, 1))
    q.copy_(torch.randn(3, 2, 256, device=DEV, generator=g))
    kv = torch.randn(2, 3, 1, 256, device=DEV, generator=g).bfloat16()
    freq, pos = FREQ.float().to(DEV), torch.tensor([0, 5, 99], device=DEV)
    want_q, want_k = qk_norm_rope(q.contiguous(), kv[0], pos, freq)
    assert torch.equal(qk_norm_rope(q, kv[0], pos, freq)[0], want_q)
    pages = (4 << 30) // (16 * 512) + 40
    pool = PagedKVCache(pages, num_layers=1, kv_heads=1, dtype=torch.bfloat16, device=DEV,
                        verbose=False)
    slots = torch.tensor([1, (pages - 20) * 16 + 7, pages * 16 - 1], device=DEV)
    assert torch.equal(pool.append_rope(slots, q, kv[0], kv[1], 0, pos, freq), want_q)
    pool.check_errors()
    rows = pool.cache.view(2, pages * 16, 1, 256)
    assert torch.equal(rows[0][slots], want_k) and torch.equal(rows[1][slots], kv[1])


@pytest.mark.parametrize("dim,tokens", [(64, 40000), (128, 33333)])
def test_many_tokens(dim, tokens):
    case(f"norm + rotation of {tokens} tokens, heads of {dim}")
    g = torch.Generator(device=DEV).manual_seed(dim)
    q, k = (torch.randn(tokens, h, dim, device=DEV, generator=g).half() for h in (3, 1))
    freq = (1e4 ** (-torch.arange(0, dim, 2).double() / dim)).to(DEV)
    pos = torch.arange(tokens, device=DEV)
    w = torch.rand(dim, device=DEV, generator=g)
    got = qk_norm_rope(q, k, pos, freq, w, w)
    angle = pos[:, None].double() * freq
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    for x, out in zip((q, k), got):
        y = x.double()
        y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        a, b = y.chunk(2, -1)
        want = torch.cat([a * c - b * s, b * c + a * s], -1)
        # a rounding to fp16 and a few of fp32, of the rotated pair's size
        size = torch.cat([a.abs() + b.abs()] * 2, -1)
        assert ((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -20 * size
                + 2.0 ** -25).all()
