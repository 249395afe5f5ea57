"""Decode attention over a 4-bit pool on both of its ways: a workgroup for each (sequence, KV
head), and spans of the list of all tiles with the kernel that joins what they cut. A wide page
table takes short sequences through the spans."""
import numpy as np
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels import attention as A
from oracle import attention as att
from oracle import fp4
from tests.gpu_util import DEV, case

pytestmark = pytest.mark.gpu

# least width of the page tables (0: the longest sequence's)
WAYS = {"pairs": 0, "spans": 600, "middle": 0, "cut": 0}


def takes(way, batch, hq, hkv, width):
    """That a call of this shape goes the way that it is meant to."""
    with torch.cuda.device(DEV):
        size = _lib.load().mkv_decode_attention_fp4_workspace_bytes(batch, hkv, hq, width * 16)
    assert (size == 0) == (way == "pairs")


def tables(rng, lens, way, spare=4):
    """Page tables over pages in no order, and the pool's pages."""
    need = [-(-int(n) // 16) for n in lens]
    pages = sum(need) + spare
    order = rng.permutation(pages)
    table = np.zeros((len(lens), max(1, WAYS[way], *need)), dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def attend(q, k, v, lens, table, **how):
    dev = [x.to(DEV) if isinstance(x, torch.Tensor) else torch.from_numpy(x).to(DEV)
           for x in (q, k, v, np.asarray(lens, dtype=np.int32), table)]
    out = A.attn_decode_fp4(*dev, **how)
    torch.cuda.synchronize()
    return out[:, 0].double().cpu().numpy()


@pytest.mark.parametrize("way", ["pairs", "spans"])
def test_probabilities_are_not_cut(way):
    """Two tokens whose weighted values nearly cancel, so that the probabilities' own errors are
    what is left. The second token's score is 0, the first one's two exact products.

    Tolerance: half a step of bf16 of what is left; of the attended mass 2^-18, a weight's second
    part rounded (the first leaves at most 2^-9 of it, of which 2^-9), and 2^-21 of fp32: three
    roundings of a score below 2 (2.1 of 2^-24), 2^x (2), the sums, the quotient and the product
    (4)."""
    case(f"4-bit decode attention, nearly cancelling values, {way}")
    rng = np.random.default_rng(21)
    B, hq = 64, 8
    table, pages = tables(rng, [2] * B, way)
    takes(way, B, hq, 1, table.shape[1])
    pairs = [(4, 3), (6, 4), (3, 2), (4, 2), (3, 1.5), (6, 3), (4, 1.5), (6, 2), (2, 1.5)]
    k, v = np.zeros((pages, 16, 1, 256)), np.zeros((pages, 16, 1, 256))
    q = torch.zeros(B, 1, hq, 256, dtype=torch.float64)
    for b in range(B):
        page = table[b, 0]
        k[page, 0, 0, 0], k[page, 0, 0, 32] = -1.0, 2.0 ** -6
        for dim in range(256):
            first, second = pairs[dim % len(pairs)]
            v[page, 0, 0, dim], v[page, 1, 0, dim] = first, -second
        for h in range(hq):
            first, second = pairs[(8 * b + h) % len(pairs)]
            score = 16 * (np.log(second / first) + rng.standard_normal() * 2.0 ** -11)
            q[b, 0, h, 0] = torch.tensor(-score, dtype=torch.float64).bfloat16().double()
            q[b, 0, h, 32] = (score + float(q[b, 0, h, 0])) * 64
    q = q.bfloat16()
    k, v = fp4.quantize_rows(k), fp4.quantize_rows(v)
    got = attend(q, k, v, [2] * B, table)
    want, mass, _ = att.decode_attention(q[:, 0].double().numpy(), fp4.values(k), fp4.values(v),
                                         [2] * B, table, 1 / 16, stats=True)
    err = np.abs(got - want)
    tol = 2.0 ** -8 * np.abs(want) + (2.0 ** -18 + 2.0 ** -21) * mass
    assert (err <= tol).all(), f"{(err > tol).sum()} of {err.size} off, worst {(err / tol).max()}"


def filled(seed, lens, hq, hkv, way, spread=1.0):
    """Queries, the two planes' rows of any codes and of scales 2^-3 to 1, page tables."""
    rng = np.random.default_rng(seed)
    table, pages = tables(rng, lens, way)
    k, v = rng.integers(0, 256, (2, pages, 16, hkv, fp4.ROW), dtype=np.uint8)
    for x in (k, v):
        x[..., 128:] = rng.integers(124, 128, x[..., 128:].shape)
    q = (spread * torch.randn(len(lens), 1, hq, 256,
                              generator=torch.Generator().manual_seed(seed))).bfloat16()
    return q, k, v, np.asarray(lens), table


@pytest.mark.parametrize("most", [1 << 25, (1 << 31) - 1, 1 << 31, 1 << 32, (1 << 32) + 5, 1 << 70])
@pytest.mark.parametrize("way", ["pairs", "spans"])
def test_bounds_that_pass_32_bits(way, most):
    """No bound at all, as without one."""
    case(f"decode attention, max_seqlen {most}, {way}")
    args = filled(22, [70, 1, 33], 4, 1, way)
    takes(way, 3, 4, 1, args[-1].shape[1])
    want = attend(*args)
    got = attend(*args, max_seqlen=most)
    A.check_errors(DEV)
    assert np.array_equal(got, want) and want.any(-1).all()
    q, k, v, lens, table = args
    dev = [x.to(DEV) for x in (q, *(torch.from_numpy(fp4.values(x)).bfloat16() for x in (k, v)),
                               torch.from_numpy(lens.astype(np.int32)), torch.from_numpy(table))]
    want = A.attn_decode(*dev)
    got = A.attn_decode(*dev, max_seqlen=most)
    A.check_errors(DEV)
    assert torch.equal(got, want) and want.any(-1).all()


# short sequences on both ways, and longer ones, which spans and workgroups cut: joined by 4
# waves ("middle") and by 16 ("cut")
SHAPES = {"pairs": [50, 60, 70, 0, 200, 17], "spans": [50, 60, 70, 0, 200, 17],
          "middle": [1500, 33, 0, 900, 1600, 17], "cut": [70000, 33, 0, 9000, 2500, 17]}


def way_of(shape):
    return "pairs" if shape == "pairs" else "spans"


def prepared(seed, shape, hq, hkv, **how):
    args = filled(seed, SHAPES[shape], hq, hkv, shape, **how)
    takes(way_of(shape), len(args[3]), hq, hkv, args[4].shape[1])
    return args


def oracle(q, k, v, lens, table, scale=1 / 16):
    return att.decode_attention(q[:, 0].double().numpy(), fp4.values(k), fp4.values(v), lens, table,
                                scale, stats=True)


def bound(want):
    """What an output may be off: half a step of bf16; of the attended mass 2^-18 of its weights'
    two parts, and 2^-16 (1 + max |score|) of the scores' sums in fp32. Below 2^-126 fp32 and bf16
    have no normal values: a weight, its second part and the output may each lose so much. With
    values up to 6, a sum of weights of 1 or more and n tokens that is at most
    (2 * 6 n + 1) 2^-126, below 2^-105 for the longest sequences here (n < 2^17)."""
    out, mass, smax = want
    return (2.0 ** -8 * np.abs(out) + (2.0 ** -18 + 2.0 ** -16 * (1 + smax[..., None])) * mass
            + 2.0 ** -105)


def close(got, want, where=None):
    err, tol = np.abs(got - want[0]), bound(want)
    bad = ~(err <= tol) if where is None else ~(err <= tol) & where
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {(err / (tol + 1e-300))[bad].max()}"


@pytest.mark.parametrize("hq,hkv", [(4, 1), (3, 1), (16, 2)])
@pytest.mark.parametrize("shape", SHAPES)
def test_values(shape, hq, hkv):
    case(f"4-bit decode attention, {shape}, {hq} heads on {hkv}")
    args = prepared(23, shape, hq, hkv)
    got = attend(*args)
    A.check_errors(DEV)
    close(got, oracle(*args))
    assert np.array_equal(got, attend(*args))  # and the same again


@pytest.mark.parametrize("spread,scale", [(40.0, None), (1e-3, None), (1.0, 3.0), (1.0, -0.5)])
@pytest.mark.parametrize("shape", ["spans", "middle", "cut"])
def test_sharp_and_flat_softmaxes(shape, spread, scale):
    case(f"4-bit decode attention, {shape}, queries x {spread}, scale {scale}")
    args = prepared(24, shape, 4, 1, spread=spread)
    close(attend(*args, softmax_scale=scale), oracle(*args, 1 / 16 if scale is None else scale))


@pytest.mark.parametrize("hkv", [1, 2])
@pytest.mark.parametrize("shape", SHAPES)
def test_what_lies_behind_a_sequence_is_not_read(shape, hkv):
    case(f"4-bit decode attention, {shape}, NaN behind the sequences' ends, {hkv} KV heads")
    q, k, v, lens, table = prepared(25, shape, 4, hkv)
    want = oracle(q, k, v, lens, table)
    used = np.zeros(k.shape[:2], dtype=bool)
    for b, n in enumerate(lens):
        at = np.arange(n)
        used[table[b][at // 16], at % 16] = True
    for x in (k, v):
        x[~used] = 0x77
        x[~used, :, 128:] = 255
    got = attend(q, k, v, lens, table)
    A.check_errors(DEV)
    close(got, want)


def test_many_short_sequences_in_the_spans():
    """Every span starts, ends and changes sequences inside a tile; NaN in all other places."""
    case("4-bit decode attention, 900 short sequences by spans, NaN behind their ends")
    lens = ([1, 17, 40, 0, 100, 31, 33, 32, 16] * 100)
    q, k, v, lens, table = filled(26, lens, 4, 1, "spans")
    takes("spans", len(lens), 4, 1, table.shape[1])
    want = oracle(q, k, v, lens, table)
    used = np.zeros(k.shape[:2], dtype=bool)
    for b, n in enumerate(lens):
        at = np.arange(n)
        used[table[b][at // 16], at % 16] = True
    for x in (k, v):
        x[~used, :, 128:] = 255
    got = attend(q, k, v, lens, table)
    A.check_errors(DEV)
    close(got, want)


# tokens of sequence 0 that hold a NaN: one, a tile, several workgroups' spans of the long one, all
STRETCHES = [(3, 4), (32, 64), (0, 48), (1024, 30000), (0, 70000)]


@pytest.mark.parametrize("first,last", STRETCHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_a_nan_stays_in_its_sequence_and_head(shape, first, last):
    case(f"4-bit decode attention, {shape}, NaN in tokens {first} to {last}")
    q, k, v, lens, table = prepared(27, shape, 4, 2)
    want = oracle(q, k, v, lens, table)
    n = int(lens[0])
    at = np.arange(min(first, n - 1), min(last, n))
    page, row = table[0][at // 16], at % 16
    k[page, row, 1, 130] = 255                    # sequence 0, KV head 1: its scores
    v[page, row, 0, 129] = 255                    # and KV head 0, dims 32 .. 63: values
    got = attend(q, k, v, lens, table)
    A.check_errors(DEV)
    bad = np.zeros(got.shape, dtype=bool)
    bad[0, 2:] = True
    bad[0, :2, 32:64] = True
    assert np.array_equal(np.isnan(got), bad)
    close(got, want, ~bad)


# pages of the sequence that are not in the pool: one, a tile's, several spans', all
PAGES = [(1, 2), (2, 4), (0, 3), (10, 90), (64, 2000), (0, 4375)]


@pytest.mark.parametrize("first,last", PAGES)
@pytest.mark.parametrize("shape", SHAPES)
def test_pages_outside_the_pool(shape, first, last):
    """Their tokens are left out, wherever spans cut the sequence, and the call is flagged."""
    case(f"4-bit decode attention, {shape}, pages {first} to {last} outside the pool")
    q, k, v, lens, table = prepared(28, shape, 4, 2)
    have = -(-int(lens[0]) // 16)
    first, last = min(first, have - 1), min(last, have)
    gone = np.arange(first, last)
    bad = table.copy()
    bad[0, gone] = np.array([len(k), -1, 2 ** 31 - 1, -2 ** 31])[gone % 4]
    got = attend(q, k, v, lens, bad)
    with pytest.raises(_lib.MkvDeviceError, match="page id"):
        A.check_errors(DEV)
    kept = np.delete(np.arange(have), gone)
    table[0, :len(kept)] = table[0, kept]
    held = lens.copy()
    held[0] = max(0, 16 * len(kept) - (16 * have - int(lens[0]) if last < have else 0))
    close(got, oracle(q, k, v, held, table))
    if len(kept) == 0:
        assert not got[0].any()


@pytest.mark.parametrize("shape", SHAPES)
def test_lengths_outside_the_table(shape):
    case(f"4-bit decode attention, {shape}, lengths beyond the table and below 0")
    q, k, v, lens, table = prepared(29, shape, 4, 1)
    holds = table.shape[1] * 16
    for b, n in ((5, holds + 1), (1, -3), (4, 2 ** 31 - 1), (0, -2 ** 31)):
        wrong = lens.copy()
        wrong[b] = n
        full = table.copy()
        full[b] = np.arange(table.shape[1]) % len(k)
        got = attend(q, k, v, wrong, full)
        with pytest.raises(_lib.MkvDeviceError, match="block table"):
            A.check_errors(DEV)
        wrong[b] = min(max(n, 0), holds)
        close(got, oracle(q, k, v, wrong, full))
    most = int(lens.max()) - 21
    got = attend(q, k, v, lens, table, max_seqlen=most)
    with pytest.raises(_lib.MkvDeviceError, match="block table"):
        A.check_errors(DEV)
    close(got, oracle(q, k, v, np.minimum(lens, most), table))


@pytest.mark.parametrize("hkv", [1, 2])
@pytest.mark.parametrize("shape", SHAPES)
def test_shared_pages_give_the_same(shape, hkv):
    case(f"4-bit decode attention, {shape}, shared pages, {hkv} KV heads")
    q, k, v, lens, table = prepared(30, shape, 4, hkv)
    many = -(-int(lens.min(where=lens > 30, initial=10 ** 6)) // 16)
    table[lens > 30, :many] = table[0, :many]
    want = oracle(q, k, v, lens, table)
    plain = attend(q, k, v, lens, table)
    close(plain, want)
    for shared in (1, len(k) // 2, len(k), 1 << 40):
        assert np.array_equal(attend(q, k, v, lens, table, shared_pages=shared), plain)
    A.check_errors(DEV)


@pytest.mark.parametrize("shape", SHAPES)
def test_in_place_and_through_a_view_of_a_table(shape):
    """The queries overwritten, also where their pieces are joined later; a table's rows apart."""
    case(f"4-bit decode attention, {shape}, in place, a view of a wider table")
    q, k, v, lens, table = prepared(31, shape, 4, 2)
    want = attend(q, k, v, lens, table)
    wide = torch.full((len(lens), table.shape[1] + 9), -7, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = torch.from_numpy(table)
    x = q.to(DEV)
    back = A.attn_decode_fp4(x, torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV),
                             torch.from_numpy(lens.astype(np.int32)).to(DEV),
                             wide[:, :table.shape[1]], out=x)
    torch.cuda.synchronize()
    A.check_errors(DEV)
    assert back is x and np.array_equal(x[:, 0].double().cpu().numpy(), want)


@pytest.mark.parametrize("shape", SHAPES)
def test_replayed_graphs(shape):
    """One capture, replayed for other lengths, queries and pages, with eager calls between."""
    case(f"4-bit decode attention, {shape}, captured and replayed")
    sets = [prepared(32 + i, shape, 4, 1) for i in range(3)]
    buf = [torch.empty_like(x if isinstance(x, torch.Tensor) else torch.from_numpy(np.asarray(x)),
                            device=DEV) for x in sets[0]]
    buf[3] = torch.zeros(len(sets[0][3]), dtype=torch.int32, device=DEV)
    buf[4].zero_()
    A.attn_decode_fp4(*buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = A.attn_decode_fp4(*buf)
    for i in (0, 1, 2, 0):
        q, k, v, lens, table = sets[i]
        lens = lens.copy()
        lens[i] = max(0, lens[i] - 5 * i)
        for b, x in zip(buf, (q, k, v, lens.astype(np.int32), table)):
            b.copy_(x if isinstance(x, torch.Tensor) else torch.from_numpy(x))
        graph.replay()
        got = out[:, 0].double().cpu().numpy()
        assert np.array_equal(got, A.attn_decode_fp4(*buf)[:, 0].double().cpu().numpy())
        A.check_errors(DEV)
        close(got, oracle(q, k, v, lens, table))


def test_pages_behind_4_gib_by_spans():
    case("4-bit decode attention by spans: pages behind 4 GiB of a plane")
    pages = (1 << 32) // (16 * fp4.ROW) + 400
    q, k, v, lens, table = filled(35, [200, 77, 0, 3100], 4, 1, "spans")
    first = pages - len(k)
    big = [torch.zeros(pages, 16, 1, fp4.ROW, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for b, x in zip(big, (k, v)):
        b[first:] = torch.from_numpy(x).to(DEV)
    takes("spans", 4, 4, 1, table.shape[1])
    for shared in (0, pages):
        got = A.attn_decode_fp4(q.to(DEV), *big, torch.from_numpy(lens.astype(np.int32)).to(DEV),
                                torch.from_numpy(table + first).to(DEV), shared_pages=shared)
        torch.cuda.synchronize()
        A.check_errors(DEV)
        close(got[:, 0].double().cpu().numpy(), oracle(q, k, v, lens, table))
    del big
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", SHAPES)
def test_scores_of_minus_infinity(shape):
    """Where all of a head's scores are -inf the softmax is NaN, not the zeros of no tokens;
    where some are, they have no weight. Pages outside the pool count as no tokens all the same."""
    case(f"4-bit decode attention, {shape}, scores of -inf")
    q, k, v, lens, table = prepared(36, shape, 4, 2)
    big = float(torch.finfo(torch.bfloat16).max)
    k[..., :32] &= 0x77                          # dims 0 .. 63 not below 0,
    k[..., :2] |= 0x77                             # dims 0 .. 3 the largest value, 6 * 2^e
    q[0, 0, 0, 0] = -torch.inf                     # heads 0, 1 of sequence 0: an infinity,
    q[0, 0, 1, :4] = -big                          # sums that pass fp32's range
    q[4, 0, 2, 1] = -torch.inf                     # head 2 of sequence 4, on KV head 1
    want = oracle(q.nan_to_num(), k, v, lens, table)
    got = attend(q, k, v, lens, table)
    A.check_errors(DEV)
    bad = np.zeros(got.shape, dtype=bool)
    bad[0, :2] = bad[4, 2] = True
    assert np.array_equal(np.isnan(got), bad)
    close(got, want, ~bad)
    # some tokens of sequence 0 keep finite scores: heads as without the others
    n = int(lens[0])
    for kept in (np.arange(n - 1, n), np.arange(0, n, 7), np.arange(n // 2, n // 2 + 33)):
        some = k.copy()
        kept = kept[kept < n]
        some[table[0][kept // 16], kept % 16, :, :2] = 0
        q[0, 0, 0] = q[0, 0, 1]
        got = attend(q, some, v, lens, table)
        bad[0] = False
        assert np.array_equal(np.isnan(got), bad)
        close(got[0, :2], tuple(x[0, :2] for x in alone(q, some, v, table, kept)))
    gone = table.copy()
    gone[0] = len(k)
    got = attend(q, k, v, lens, gone)
    with pytest.raises(_lib.MkvDeviceError, match="page id"):
        A.check_errors(DEV)
    assert not got[0].any()


def alone(q, k, v, table, kept):
    """The oracle over sequence 0's tokens ``kept``: the others' weights are exp(-inf)."""
    page, row = table[0][kept // 16], kept % 16
    pages = -(-len(kept) // 16)
    packed = np.zeros((2, pages * 16, *k.shape[2:]), dtype=np.uint8)
    packed[0, :len(kept)], packed[1, :len(kept)] = k[page, row], v[page, row]
    packed = packed.reshape(2, pages, 16, *k.shape[2:])
    return oracle(q[:1], packed[0], packed[1], [len(kept)], np.arange(pages)[None])
