"""The 4-bit pool: append bit-exact against the oracle, the gather's values equal to it,
page copies and the host tier."""
import numpy as np
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kv_cache import PagedKVCache
from muserve_amd.memory.host_tier import HostTier
from oracle import fp4
from tests.gpu_util import DEV, bits16, case

pytestmark = pytest.mark.gpu
FP4 = torch.float4_e2m1fn_x2


def make_pool(pages, layers=1, heads=1):
    return PagedKVCache(pages, num_layers=layers, kv_heads=heads, dtype=FP4, device=DEV,
                        verbose=False)


def rows_of(x: torch.Tensor) -> torch.Tensor:
    return torch.from_numpy(fp4.quantize_rows(x.double().numpy()))


def special_rows(heads):
    rows = torch.zeros(12, heads, 256)
    rows[1] = -0.0
    rows[2, :, 5] = 3.3895313892515355e38          # the largest bf16
    rows[3] = torch.linspace(-1e-38, 1e-38, 256)    # bf16 subnormals
    rows[4] = 1.0
    rows[4, :, 0] = -1.0
    rows[5] = torch.arange(256) * 1e-3
    rows[6] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 32)  # ties
    rows[7, :, ::2] = -7.0
    rows[8, :, 3] = float("inf")
    rows[9, :, 100] = float("nan")
    rows[10] = torch.tensor([7.0, 7.03125, 6.96875, -7.0] * 64)
    rows[11] = 2.0 ** -121
    return rows.bfloat16()


@pytest.mark.parametrize("heads", [1, 2, 3])
def test_append_is_bit_exact(heads):
    case(f"4-bit append, {heads} heads")
    g = torch.Generator().manual_seed(heads)
    pages, layers, T = 40, 2, 333
    cache = make_pool(pages, layers, heads)
    cache.cache.fill_(0x5A)
    slots = torch.randperm(pages * 16, generator=g)[:T]
    k, v = (torch.randn(layers, T, heads, 256, generator=g).bfloat16() for _ in range(2))
    k[0, :12], v[1, 3:15] = special_rows(heads), special_rows(heads)
    cache.append(slots.to(DEV), k.to(DEV), v.to(DEV))
    cache.check_errors()
    want = torch.full((layers, 2, pages * 16, heads, fp4.ROW), 0x5A, dtype=torch.uint8)
    for l in range(layers):
        want[l, 0, slots], want[l, 1, slots] = rows_of(k[l]), rows_of(v[l])
    assert torch.equal(cache.cache.cpu().view_as(want), want)


@pytest.mark.parametrize("exponent", [-126, -121, -118, -60, -3, 0, 1, 64, 125, 127])
def test_every_bf16_value_below_a_blocks_largest(exponent):
    """All bf16 values up to 1.75 and up to 1.875 times 2^exponent, signs included, in blocks
    whose largest one that is."""
    case(f"4-bit append, values below 2^{exponent + 1}")
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    every = bits.view(torch.bfloat16)
    rows = []
    for most in (1.75, 1.875):
        top = torch.tensor(most * 2.0 ** exponent).bfloat16()
        x = every[every.abs() <= top]
        x = torch.nn.functional.pad(x, (0, -len(x) % 31)).view(-1, 31)
        x = torch.cat([x, top.expand(len(x), 1)], 1).flatten()
        rows.append(torch.nn.functional.pad(x, (0, -len(x) % 256)).view(-1, 1, 256))
    x = torch.cat(rows)
    cache = make_pool(-(-len(x) // 16))
    slots = torch.arange(len(x), device=DEV)
    cache.append(slots, x.to(DEV), x.to(DEV), layer=0)
    cache.check_errors()
    want = rows_of(x)
    for plane in range(2):
        got = cache.cache[0, plane].reshape(-1, 1, fp4.ROW)[:len(x)].cpu()
        assert torch.equal(got, want)


def test_skipped_and_bad_slots():
    case("4-bit append: slot -1 and slots outside the pool")
    g = torch.Generator().manual_seed(5)
    cache = make_pool(4, heads=2)
    x = torch.randn(3, 2, 256, generator=g).bfloat16()
    cache.append(torch.tensor([5, -1, 63], device=DEV), x.to(DEV), x.to(DEV), layer=0)
    cache.check_errors()
    want = torch.zeros(64, 2, fp4.ROW, dtype=torch.uint8)
    want[[5, 63]] = rows_of(x[[0, 2]])
    assert torch.equal(cache.cache[0, 0].view(64, 2, fp4.ROW).cpu(), want)
    for bad in (64, -2, 1 << 40):
        cache.append(torch.tensor([7, bad], device=DEV), x[:2].to(DEV), x[:2].to(DEV), layer=0)
        with pytest.raises(_lib.MkvDeviceError, match="slot_mapping"):
            cache.check_errors()
    want[7] = rows_of(x[:1])[0]
    assert torch.equal(cache.cache[0, 1].view(64, 2, fp4.ROW).cpu(), want)


def filled(pages, layers, heads, seed):
    """A pool of quantised normal values, and its values by [layer, plane, slot]."""
    cache = make_pool(pages, layers, heads)
    x = torch.randn(layers, 2, pages * 16, heads, 256,
                    generator=torch.Generator().manual_seed(seed)).bfloat16()
    slots = torch.arange(pages * 16, device=DEV)
    cache.append(slots, x[:, 0].to(DEV), x[:, 1].to(DEV))
    cache.check_errors()
    value = torch.from_numpy(fp4.values(rows_of(x).numpy()))
    assert torch.equal(value, value.bfloat16().double())  # values of the pool are bf16 values
    return cache, value.bfloat16()


def tables_of(rng, lens, pages, width=None):
    need = [-(-int(n) // 16) for n in lens]
    order = rng.permutation(pages)
    table = np.zeros((len(lens), width or max(1, max(need))), dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table


def sequence(value, table_row, start, n):
    pos = torch.arange(start, start + n)
    return value[torch.from_numpy(table_row.astype(np.int64))[pos // 16] * 16 + pos % 16]


LENS = [1, 15, 16, 17, 0, 33, 64, 100, 47]


@pytest.mark.parametrize("heads", [1, 2, 3, 5])
@pytest.mark.parametrize("out_len", [48, 100, 113])
def test_padded_gather(heads, out_len):
    case(f"4-bit gather padded, {heads} heads, {out_len} rows")
    rng = np.random.default_rng(heads)
    cache, value = filled(40, 2, heads, 11)
    table = tables_of(rng, LENS, 40)
    starts = np.array([0, 3, 15, 0, 0, 31, 16, 40, 50], dtype=np.int32)
    lens = torch.tensor(LENS, dtype=torch.int32, device=DEV)
    for st in (None, starts):
        k, v = cache.gather(None, torch.from_numpy(table).to(DEV), lens, out_len=out_len,
                            starts=None if st is None else torch.from_numpy(st).to(DEV))
        cache.check_errors()
        for l in range(2):
            for plane, got in ((0, k), (1, v)):
                want = torch.zeros(len(LENS), out_len, heads, 256, dtype=torch.bfloat16)
                for b, n in enumerate(LENS):
                    s = 0 if st is None else int(st[b])
                    m = max(0, min(n - s, out_len))
                    want[b, :m] = sequence(value[l, plane], table[b], s, m)
                assert torch.equal(bits16(got[l]), bits16(want))


@pytest.mark.parametrize("heads", [1, 2, 3])
def test_packed_gather_leaves_other_rows(heads):
    case(f"4-bit gather packed, {heads} heads")
    rng = np.random.default_rng(heads)
    cache, value = filled(40, 1, heads, 12)
    table = tables_of(rng, LENS, 40)
    gaps = np.concatenate([[2], 2 + np.cumsum(np.array(LENS) + 1)])
    cu = torch.from_numpy(gaps.astype(np.int64)).to(DEV)
    total = int(gaps[-1]) + 5
    out = tuple(torch.full((total, heads, 256), 7.0, dtype=torch.bfloat16, device=DEV)
                for _ in range(2))
    cache.gather(0, torch.from_numpy(table).to(DEV),
                 torch.tensor(LENS, dtype=torch.int32, device=DEV), out_len=100, cu_out=cu, out=out)
    cache.check_errors()
    for plane in range(2):
        want = torch.full((total, heads, 256), 7.0, dtype=torch.bfloat16)
        for b, n in enumerate(LENS):
            want[gaps[b]:gaps[b] + n] = sequence(value[0, plane], table[b], 0, n)
        assert torch.equal(bits16(out[plane]), bits16(want))


def test_gather_of_bad_pages_and_long_sequences():
    case("4-bit gather: page ids outside the pool, lengths beyond the table")
    cache, value = filled(6, 1, 2, 13)
    for bad in (6, -1, 2 ** 31 - 1):
        table = torch.tensor([[3, bad, 1]], dtype=torch.int32)
        k, _ = cache.gather(0, table.to(DEV), torch.tensor([40], dtype=torch.int32, device=DEV),
                            out_len=48)
        with pytest.raises(_lib.MkvDeviceError, match="page id"):
            cache.check_errors()
        want = torch.zeros(1, 48, 2, 256, dtype=torch.bfloat16)
        want[0, :16], want[0, 32:40] = value[0, 0, 48:64], value[0, 0, 16:24]
        assert torch.equal(bits16(k), bits16(want))
    k, _ = cache.gather(0, torch.tensor([[5]], dtype=torch.int32, device=DEV),
                        torch.tensor([20], dtype=torch.int32, device=DEV), out_len=32)
    with pytest.raises(_lib.MkvDeviceError, match="block table"):
        cache.check_errors()
    assert torch.equal(bits16(k[0, :16]), bits16(value[0, 0, 80:]))
    assert not k[0, 16:].any()


def test_nan_blocks_and_rows_never_written():
    case("4-bit gather: NaN blocks, rows never written")
    cache = make_pool(2)
    x = special_rows(1)
    cache.append(torch.arange(12, device=DEV), x.to(DEV), x.to(DEV), layer=0)
    k, _ = cache.gather(0, torch.tensor([[0, 1]], dtype=torch.int32, device=DEV),
                        torch.tensor([32], dtype=torch.int32, device=DEV))
    cache.check_errors()
    got = k[0, :, 0].cpu().double()
    want = torch.zeros(32, 256, dtype=torch.float64)
    want[:12] = torch.from_numpy(fp4.values(rows_of(x[:, 0]).numpy()))
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_write_kv_copy_pages_and_the_host_tier():
    case("4-bit write_kv, copy_pages, host tier")
    g = torch.Generator().manual_seed(9)
    cache = make_pool(8, 2, 1)
    x = torch.randn(16, 1, 256, generator=g).bfloat16()
    cache.write_kv(1, 3, slice(0, 16), x.to(DEV), x.to(DEV))
    assert torch.equal(cache.cache[1, 0, 3].cpu(), rows_of(x))
    k, v = cache.get_kv_by_layer(1)
    assert k.shape == (8, 16, 1, fp4.ROW) and torch.equal(k[3], v[3])
    cache.copy_pages([3], [6])
    cache.check_errors()
    assert torch.equal(cache.cache[:, :, 6], cache.cache[:, :, 3])
    tier = HostTier(1 << 20, DEV)
    held = tier.put_blocks(cache.cache, 3, torch.tensor([3, 6]))
    before = cache.cache.clone()
    cache.cache.zero_()
    tier.get_blocks(held, cache.cache, 3, torch.tensor([3, 6]))
    tier.check_errors()
    torch.cuda.synchronize()
    assert torch.equal(cache.cache, before)


def test_rows_behind_4_gib():
    case("4-bit append and gather behind 4 GiB of a plane")
    pages = (1 << 32) // (16 * fp4.ROW) + 40
    cache = make_pool(pages)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(20, 1, 256, generator=g).bfloat16()
    last = pages * 16 - 20
    cache.append(torch.arange(last, last + 20, device=DEV), x.to(DEV), (-x).to(DEV), layer=0)
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device=DEV)
    k, v = cache.gather(0, table, torch.tensor([32], dtype=torch.int32, device=DEV))
    cache.check_errors()
    want = torch.from_numpy(fp4.values(rows_of(x).numpy()))[:, 0]
    assert torch.equal(k[0, 12:, 0].cpu().double(), want)
    assert torch.equal(v[0, 12:, 0].cpu().double(), -want)
    del cache, k, v
    torch.cuda.empty_cache()


def test_appends_and_gathers_in_a_graph():
    case("4-bit append and gather captured, replayed")
    g = torch.Generator().manual_seed(3)
    cache = make_pool(8, 1, 2)
    x = torch.empty(40, 2, 256, dtype=torch.bfloat16, device=DEV)
    slots = torch.empty(40, dtype=torch.int64, device=DEV)
    table = torch.tensor([[2, 5, 1]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([48], dtype=torch.int32, device=DEV)
    out = tuple(torch.empty(1, 48, 2, 256, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    x.zero_()
    slots.fill_(-1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.append(slots, x, x, layer=0)
        cache.gather(0, table, lens, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(slots, x, x, layer=0)
        cache.gather(0, table, lens, out=out)
    for _ in range(3):
        fresh = torch.randn(40, 2, 256, generator=g).bfloat16()
        at = torch.randperm(128, generator=g)[:40]
        x.copy_(fresh)
        slots.copy_(at)
        want = cache.cache[0, 0].view(128, 2, fp4.ROW).cpu()
        want[at] = rows_of(fresh)
        graph.replay()
        torch.cuda.synchronize()
        cache.check_errors()
        assert torch.equal(cache.cache[0, 0].view(128, 2, fp4.ROW).cpu(), want)
        values = torch.from_numpy(fp4.values(want.view(8, 16, 2, fp4.ROW)[[2, 5, 1]].numpy()))
        assert torch.equal(out[1][0].cpu().double(), values.flatten(0, 1))
