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

WAYS = {"pairs": 0, "spans": 600}  # least width of the page tables (0: the longest sequence's)


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


@pytest.mark.parametrize("way", WAYS)
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
    """Queries, the two planes' rows of quantised normal values, page tables."""
    rng, g = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    table, pages = tables(rng, lens, way)
    k, v = (fp4.quantize_rows(torch.randn(pages, 16, hkv, 256, generator=g).bfloat16().double().numpy())
            for _ in range(2))
    q = (spread * torch.randn(len(lens), 1, hq, 256, generator=g)).bfloat16()
    return q, k, v, np.asarray(lens), table


@pytest.mark.parametrize("most", [1 << 25, (1 << 31) - 1, 1 << 31, 1 << 32, (1 << 32) + 5, 1 << 70])
@pytest.mark.parametrize("way", WAYS)
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
