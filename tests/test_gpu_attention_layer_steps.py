"""A 4-bit pool's steps as a serving loop makes them: bounds and windows from the plan's host
side, the windows packed into kept buffers; the packed gather captured and replayed."""
import itertools

import numpy as np
import pytest
import torch

from muserve_amd.kernels import attention as A
from muserve_amd.kv_cache import PagedKVCache
from muserve_amd.scheduler import ContinuousBatchScheduler, InferenceRequest
from oracle import attention as att
from oracle import fp4
from tests.gpu_util import DEV, bits16, case

pytestmark = pytest.mark.gpu
POOLS = [torch.bfloat16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2]


def make_pool(pages, dtype=torch.float4_e2m1fn_x2, heads=1):
    return PagedKVCache(pages, num_layers=1, kv_heads=heads, dtype=dtype, device=DEV, verbose=False)


def test_steps_with_bounds_from_the_plan():
    """Lengths and windows that the host knows are those that the device has, and the calls made
    with them attend to what the oracle does."""
    case("4-bit pool: steps with the plan's own bounds")
    rng, g = np.random.default_rng(6), torch.Generator(device=DEV).manual_seed(6)
    hq, hk, layer = 4, 1, 0
    cache = make_pool(512)
    s = ContinuousBatchScheduler(max_batch_size=5, max_seq_len=2048, kv_cache=cache,
                                 chunked_prefill_size=256)
    for i, n in enumerate([30, 1500, 5, 700, 40, 90, 1100, 3]):
        s.add_request(InferenceRequest(request_id=str(i), input_ids=list(range(n)),
                                       max_new_tokens=int(rng.integers(3, 14))))
    inv_freq = (1e6 ** (-torch.arange(0, 64, 2).double() / 64)).float().to(DEV)
    buffers = [torch.zeros(2048 * 5, hk, 256, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    mixed = 0
    while (plan := s.plan_step()) is not None:
        nd, lens = plan.num_decode, plan.seq_lens.tolist()
        longest_decode = max((r.total_len for r in plan.decode), default=0)
        windows = [start + count for _, start, count in plan.prefill]
        assert [r.total_len for r in plan.decode] + windows == lens
        cu = torch.tensor([0, *itertools.accumulate(windows)], device=cache.device)
        k_buf, v_buf = (b[:sum(windows)] for b in buffers)
        x = torch.randn(plan.num_tokens, (hq + 2 * hk) * 256, device=DEV, generator=g).bfloat16()
        q, k, v = (y.unflatten(1, (-1, 256)) for y in x.split([hq * 256, hk * 256, hk * 256], 1))
        q = cache.append_rope(plan.slot_mapping, q, k, v, layer, plan.positions, inv_freq)
        table = plan.block_tables.cpu().numpy()
        if nd:
            out = A.attn_decode_fp4(q[:nd, None], *cache.get_kv_by_layer(layer), plan.seq_lens[:nd],
                                    plan.block_tables[:nd], max_seqlen=longest_decode)
        if windows:
            k_win, v_win = cache.gather(layer, plan.block_tables[nd:], plan.seq_lens[nd:],
                                        out_len=max(windows), cu_out=cu, out=(k_buf, v_buf))
        cache.check_errors()
        A.check_errors(DEV)
        if nd and windows and mixed < 8:
            mixed += 1
            kc, vc = (fp4.values(y.cpu().numpy()) for y in cache.get_kv_by_layer(layer))
            want, mass, smax = att.decode_attention(q[:nd].double().cpu().numpy(), kc, vc,
                                                    np.array(lens[:nd]), table[:nd], 1 / 16, stats=True)
            tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -18 + 2.0 ** -16 * (1 + smax[..., None])) * mass
            assert (np.abs(out[:, 0].double().cpu().numpy() - want) <= tol).all()
            for got, pool in ((k_win, kc), (v_win, vc)):
                rows = np.concatenate([att.gather_kv(pool, t, n) for t, n in zip(table[nd:], windows)])
                assert np.array_equal(got.double().cpu().numpy(), rows)
        s.complete_step(plan, rng.integers(4, 64, len(plan.entries)).tolist())
    assert mixed >= 5


@pytest.mark.parametrize("dtype", POOLS)
def test_a_packed_gather_in_a_graph(dtype):
    """Captured with buffers given; replayed for other windows and pages, with eager calls between."""
    case(f"packed gather captured, pool of {dtype}")
    g = torch.Generator().manual_seed(7)
    cache = make_pool(40, dtype, heads=2)
    x = torch.randn(2, 640, 2, 256, generator=g).bfloat16().to(DEV)
    cache.append(torch.arange(640, device=DEV), x[0], x[1], layer=0)
    table = torch.zeros(3, 12, dtype=torch.int32, device=DEV)
    lens, starts = (torch.zeros(3, dtype=torch.int32, device=DEV) for _ in range(2))
    cu = torch.zeros(4, dtype=torch.int64, device=DEV)
    out, eager = ([torch.full((500, 2, 256), 7.0, dtype=torch.bfloat16, device=DEV)
                   for _ in range(2)] for _ in range(2))

    def gather(to):
        cache.gather(0, table, lens, out_len=192, starts=starts, cu_out=cu, out=tuple(to))

    gather(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gather(out)
    for lengths, first in (([100, 0, 33], [0, 0, 5]), ([1, 192, 16], [0, 30, 0]),
                           ([190, 64, 17], [100, 64, 16]), ([0, 0, 0], [0, 0, 0])):
        table.copy_(torch.randperm(40, generator=g)[:36].view(3, 12))
        lens.copy_(torch.tensor(lengths))
        starts.copy_(torch.tensor(first))
        cu.copy_(torch.tensor([2, *itertools.accumulate(n - f + 1 for n, f in zip(lengths, first))]))
        cu[1:] += 2
        for y in (*out, *eager):
            y.fill_(7.0)
        graph.replay()
        gather(eager)
        torch.cuda.synchronize()
        cache.check_errors()
        for a, b in zip(out, eager):
            assert torch.equal(bits16(a), bits16(b))
        at = cu.tolist()
        for plane in range(2):
            whole = cache.gather(0, table, lens, out_len=192, starts=starts)[plane]
            want = torch.full((500, 2, 256), 7.0, dtype=torch.bfloat16, device=DEV)
            for b, n in enumerate(n - f for n, f in zip(lengths, first)):
                want[at[b]:at[b] + n] = whole[b, :n]
            assert torch.equal(bits16(out[plane]), bits16(want))
