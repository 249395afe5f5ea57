"""Decode attention over a 4-bit pool against the float64 oracle on the values that the pool
stands for.

Tolerance: one rounding to bf16 (2^-8 of the value), plus what an fp32 evaluation is off: the
scores' 256-term sums shift the weights by 2^-16 * (1 + max |score|) of the attended mass
sum_j p_j |v_j| / sum_j p_j, and the weights enter the product with V in two parts of 8
significant bits, each cut: 2^-14 of a weight (2^-7 of what 2^-7 of it left)."""
import numpy as np
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels import attention as A
from oracle import attention as att
from oracle import fp4
from tests.gpu_util import DEV, case

pytestmark = pytest.mark.gpu


def build(seed, lens, hq, hkv, spare=5, width=None, spread=1.0):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, dtype=np.int64)
    pages = [-(-int(n) // 16) for n in lens]
    P = sum(pages) + spare
    perm = rng.permutation(P)
    table = np.zeros((len(lens), width or max(1, max(pages))), dtype=np.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    g = torch.Generator().manual_seed(seed)
    k, v = (fp4.quantize_rows(torch.randn(P, 16, hkv, 256, generator=g).bfloat16().double().numpy())
            for _ in range(2))
    q = (spread * torch.randn(len(lens), 1, hq, 256, generator=g)).bfloat16()
    return q, k, v, lens, table


def close(got, want):
    out, mass, smax = want
    got = got.float().cpu().numpy().astype(np.float64)
    tol = 2.0 ** -8 * np.abs(out) + (2.0 ** -14 + 2.0 ** -16 * (1 + smax[..., None])) * mass
    err = np.abs(got - out)
    assert (err <= tol).all(), f"{(err > tol).sum()} of {err.size} off, worst {(err / (tol + 1e-300)).max()}"


def run(q, k, v, lens, table, **how):
    dev = [x.to(DEV) if isinstance(x, torch.Tensor) else torch.from_numpy(x).to(DEV)
           for x in (q, k, v, lens.astype(np.int32), table)]
    out = A.attn_decode_fp4(*dev, **how)
    torch.cuda.synchronize()
    return out[:, 0]


def oracle(q, k, v, lens, table, scale=256 ** -0.5):
    return att.decode_attention(q[:, 0].double().numpy(), fp4.values(k), fp4.values(v), lens, table,
                                scale, stats=True)


LENS = [1, 2, 15, 16, 17, 31, 32, 33, 200, 511, 512, 513, 1000, 1023, 1024, 1025, 1500, 0, 7]


@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 1), (3, 1), (4, 1), (5, 1), (8, 1), (4, 2), (6, 3),
                                    (16, 2)])
def test_matches_the_oracle(hq, hkv):
    case(f"4-bit decode attention, {hq} heads on {hkv}")
    args = build(17 * hq + hkv, LENS, hq, hkv)
    got = run(*args)
    A.check_errors(DEV)
    close(got, oracle(*args))


@pytest.mark.parametrize("lens", [
    [1], [32], [33], [4096], [16 * 127 + 5], [16 * 1200 + 1, 0, 9], [40000], [20] * 126 + [4800],
    [5] * 700, [0, 0, 0], list(range(1, 120)),
    # around the longest contexts that get a workgroup for each sequence
    [768], [784], [300, 768, 0, 31], [300, 784, 0, 31], [900] + [7] * 127, [1040] + [7] * 127,
    [20] * 512, [20] * 513])
def test_shapes_of_batches(lens):
    case(f"4-bit decode attention: {len(lens)} sequences, longest {max(lens)}")
    args = build(3 + len(lens), lens, 4, 1)
    got = run(*args)
    A.check_errors(DEV)
    close(got, oracle(*args))


@pytest.mark.parametrize("spread,scale", [(40.0, None), (1e-3, None), (1.0, 3.0), (1.0, -0.5)])
def test_sharp_and_flat_softmaxes(spread, scale):
    case(f"4-bit decode attention, queries x {spread}, scale {scale}")
    q, k, v, lens, table = build(5, [700, 64, 33], 4, 1, spread=spread)
    got = run(q, k, v, lens, table, softmax_scale=scale)
    close(got, oracle(q, k, v, lens, table, 256 ** -0.5 if scale is None else scale))


def test_rising_scores():
    """Every token's score passes the ones before it by far: the maximum rises in each tile."""
    case("4-bit decode attention, rising scores")
    n = 1500
    q, k, v, lens, table = build(6, [n], 4, 1)
    x = torch.ones(n, 1, 256, dtype=torch.float64)
    x *= 2.0 ** (torch.arange(n) // 120 - 6).double()[:, None, None]
    rows = fp4.quantize_rows(x.numpy())
    at = table[0][np.arange(n) // 16].astype(np.int64) * 16 + np.arange(n) % 16
    k.reshape(-1, 1, fp4.ROW)[at] = rows
    q = torch.full_like(q, 0.25)
    q[0, 0, 1] = -0.25  # and falls, for another head
    got = run(q, k, v, lens, table)
    close(got, oracle(q, k, v, lens, table))


def test_what_lies_behind_a_sequence_is_not_read():
    case("4-bit decode attention: NaN behind the sequences' ends")
    q, k, v, lens, table = build(7, [1, 17, 40, 100, 0], 4, 2)
    want = oracle(q, k, v, lens, table)
    used = np.zeros(k.shape[:2], dtype=bool)
    for b, n in enumerate(lens):
        pos = np.arange(n)
        used[table[b][pos // 16], pos % 16] = True
    for x in (k, v):
        x[~used] = 0x77
        x[~used, :, 128:] = 255
    got = run(q, k, v, lens, table)
    A.check_errors(DEV)
    close(got, want)


def test_a_nan_stays_in_its_sequence_and_head():
    case("4-bit decode attention: NaN values")
    q, k, v, lens, table = build(8, [50, 60, 70], 4, 2)
    want = oracle(q, k, v, lens, table)
    k[table[0, 1], 3, 1, 130] = 255      # sequence 0, KV head 1: its scores
    v[table[2, 0], 5, 0, 129] = 255      # sequence 2, KV head 0: dims 32 .. 63
    got = run(q, k, v, lens, table).float().cpu()
    bad = torch.zeros(3, 4, 256, dtype=torch.bool)
    bad[0, 2:] = True
    bad[2, :2, 32:64] = True
    assert torch.equal(got.isnan(), bad)
    keep = ~bad.numpy()
    out, mass, smax = want
    tol = 2.0 ** -8 * np.abs(out) + (2.0 ** -14 + 2.0 ** -16 * (1 + smax[..., None])) * mass
    assert (np.abs(got.numpy().astype(np.float64) - out) <= tol)[keep].all()


def test_bad_pages_and_lengths():
    case("4-bit decode attention: pages outside the pool, lengths beyond the table")
    q, k, v, lens, table = build(9, [64, 40], 4, 1)
    for bad in (len(k), -1, 2 ** 31 - 1):
        t = table.copy()
        t[0, 1] = bad
        got = run(q, k, v, lens, t)
        with pytest.raises(_lib.MkvDeviceError, match="page id"):
            A.check_errors(DEV)
        # as without the page's tokens
        t[0] = [table[0, 0], table[0, 2], table[0, 3], 0]
        close(got, oracle(q, k, v, np.array([48, 40]), t))
    got = run(q, k, v, np.array([200, -3]), table)
    with pytest.raises(_lib.MkvDeviceError, match="block table"):
        A.check_errors(DEV)
    close(got, oracle(q, k, v, np.array([64, 0]), table))
    got = run(q, k, v, lens, table, max_seqlen=33)
    with pytest.raises(_lib.MkvDeviceError, match="block table"):
        A.check_errors(DEV)
    close(got, oracle(q, k, v, np.array([33, 33]), table))


def test_shared_pages_give_the_same():
    case("4-bit decode attention: shared pages")
    q, k, v, lens, table = build(10, [300, 300, 300, 17], 4, 1)
    table[1, :10] = table[0, :10]
    table[2, :10] = table[0, :10]
    for shared in (0, 7, len(k)):
        got = run(q, k, v, lens, table, shared_pages=shared)
        A.check_errors(DEV)
        close(got, oracle(q, k, v, lens, table))


def test_strided_tables_and_given_outputs():
    case("4-bit decode attention: a view of a wider table, an output given")
    q, k, v, lens, table = build(11, [90, 5, 33], 4, 1)
    wide = torch.full((3, 40), -7, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = torch.from_numpy(table)
    out = torch.full((3, 1, 4, 256), float("nan"), dtype=torch.bfloat16, device=DEV)
    back = A.attn_decode_fp4(q.to(DEV), torch.from_numpy(k).to(DEV), torch.from_numpy(v).to(DEV),
                             torch.from_numpy(lens.astype(np.int32)).to(DEV),
                             wide[:, :table.shape[1]], out=out)
    torch.cuda.synchronize()
    A.check_errors(DEV)
    assert back is out
    close(out[:, 0], oracle(q, k, v, lens, table))


def test_two_streams_and_two_graphs():
    case("4-bit decode attention on two streams, and two graphs replayed in turn")
    sets = [build(12 + i, [1000 + 7 * i, 30, 513], 4, 1) for i in range(2)]
    dev = [[x.to(DEV) if isinstance(x, torch.Tensor) else torch.from_numpy(x).to(DEV)
            for x in (q, k, v, lens.astype(np.int32), table)] for q, k, v, lens, table in sets]
    want = [oracle(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [None, None]
    for i in (0, 1):
        with torch.cuda.stream(streams[i]):
            for _ in range(4):
                outs[i] = A.attn_decode_fp4(*dev[i])
    torch.cuda.synchronize()
    for i in (0, 1):
        close(outs[i][:, 0], want[i])
    graphs, kept = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append(A.attn_decode_fp4(*dev[i]))
        graphs.append(graph)
    for _ in range(3):
        for i in (0, 1):
            kept[i].zero_()
            with torch.cuda.stream(streams[i]):
                streams[i].wait_stream(torch.cuda.current_stream())
                graphs[i].replay()
        eager = A.attn_decode_fp4(*dev[0])
        torch.cuda.synchronize()
        for i in (0, 1):
            close(kept[i][:, 0], want[i])
        assert torch.equal(eager, kept[0])
    # another length in the same buffers
    dev[0][3].fill_(16)
    graphs[0].replay()
    torch.cuda.synchronize()
    q, k, v, _, table = sets[0]
    close(kept[0][:, 0], oracle(q, k, v, np.array([16, 16, 16]), table))


def test_pages_behind_4_gib():
    case("4-bit decode attention: pages behind 4 GiB of a plane")
    pages = (1 << 32) // (16 * fp4.ROW) + 40
    q, k, v, lens, table = build(14, [200, 77], 4, 1)
    first = pages - len(k)
    big = [torch.zeros(pages, 16, 1, fp4.ROW, dtype=torch.uint8, device=DEV) for _ in range(2)]
    for b, x in zip(big, (k, v)):
        b[first:] = torch.from_numpy(x).to(DEV)
    got = A.attn_decode_fp4(q.to(DEV), *big, torch.from_numpy(lens.astype(np.int32)).to(DEV),
                            torch.from_numpy(table + first).to(DEV))
    torch.cuda.synchronize()
    A.check_errors(DEV)
    close(got[:, 0], oracle(q, k, v, lens, table))
    del big
    torch.cuda.empty_cache()


def test_refusals():
    case("4-bit decode attention: refused arguments")
    q, k, v, lens, table = build(15, [20], 4, 1)
    dev = [x.to(DEV) if isinstance(x, torch.Tensor) else torch.from_numpy(x).to(DEV)
           for x in (q, k, v, lens.astype(np.int32), table)]

    def refused(error, at, value, **how):
        args = list(dev)
        args[at] = value
        with pytest.raises(error):
            A.attn_decode_fp4(*args, **how)

    refused(TypeError, 0, dev[0].half())
    refused(TypeError, 1, dev[1].int())
    refused(ValueError, 0, dev[0][..., :128])
    refused(ValueError, 0, dev[0].expand(1, 1, 4, 256).repeat(1, 1, 4, 1))  # 16 on one
    refused(ValueError, 0, dev[0][:, :, :3].repeat(2, 1, 1, 1))             # two sequences of q
    refused(ValueError, 1, dev[1][..., :128])
    refused(ValueError, 2, dev[2][:3])
    refused(TypeError, 3, dev[3].long())
    refused(ValueError, 3, dev[3].repeat(2))
    refused(ValueError, 4, None)
    refused(TypeError, 4, dev[4].long())
    refused(ValueError, 0, dev[0], shared_pages=-1)
    refused(ValueError, 0, dev[0], max_seqlen=-1)
    refused(ValueError, 0, dev[0], out=torch.empty(1, 1, 4, 128, device=DEV, dtype=torch.bfloat16))
    refused(RuntimeError, 0, q)
    out = A.attn_decode_fp4(dev[0][:0], dev[1], dev[2], dev[3][:0], dev[4][:0])
    assert out.shape == (0, 1, 4, 256)
