"""Arguments of the attention layer's operators that are settled before a launch: what reaches
the library, and what does not. The launches themselves are replaced, so no GPU is needed."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels import attention, rope
from muserve_amd.kv_cache import _DTYPE_MAP, PagedKVCache

ROOT = Path(__file__).resolve().parent.parent
CPU = torch.device("cpu")
FAKE = 1 << 20  # an aligned non-null address; argument checks fail before any use


@pytest.fixture
def calls(monkeypatch):
    """The launches that would have been made: (entry point, arguments)."""
    made = []
    for module, kept in ((rope, "_plans"), (attention, "_fp4_plans"), (attention, "_errors")):
        monkeypatch.setattr(module, kept, {})  # (what is kept here is of no device)
    monkeypatch.setattr(_lib, "require_gpu", lambda *tensors: CPU)
    monkeypatch.setattr(_lib, "call_on", lambda dev, name, *args: made.append((name, args)))
    monkeypatch.setattr(_lib, "call", lambda name, *args: made.append((name, args)))
    monkeypatch.setattr(_lib, "stream_of", lambda dev: 0)
    monkeypatch.setattr(PagedKVCache, "_gpu", lambda self: self.device)
    return made


def pool(dtype=torch.bfloat16, layers=1, heads=1, pages=4):
    cache = PagedKVCache(pages, num_layers=layers, kv_heads=heads, dtype=dtype, device="cpu",
                         verbose=False)
    cache._errors = _lib.DeviceErrors(CPU)
    return cache


def test_an_output_in_place_of_a_tensor_that_is_given_twice(calls):
    """q's rows are k's rows as well: written in place they are still read as k."""
    freq, pos = torch.ones(32), torch.arange(3)
    x, y = (torch.zeros(3, 1, 256, dtype=torch.bfloat16) for _ in range(2))
    for out in ((x, y), (y, x), (x, x), (y, y)):
        with pytest.raises(ValueError, match="overlaps"):
            rope.qk_norm_rope(x, x, pos, freq, out=out)
    cache, slots = pool(), torch.arange(3)
    with pytest.raises(ValueError, match="overlaps"):
        cache.append_rope(slots, x, x, y, 0, pos, freq, out=x)
    with pytest.raises(ValueError, match="overlaps"):
        cache.append_rope(slots, x, y, x, 0, pos, freq, out=x)
    assert not calls
    # what is not read by other rows stays allowed
    z = torch.zeros_like(x)
    rope.qk_norm_rope(x, x, pos, freq, out=(y, z))
    rope.qk_norm_rope(x, y, pos, freq, out=(x, y))
    cache.append_rope(slots, x, y, y, 0, pos, freq, out=x)
    assert [name for name, _ in calls] == ["mkv_qk_norm_rope"] * 2 + ["mkv_append_rope"]


BOUNDS = [(None, 64), (40, 40), (64, 64), (65, 64), (1 << 25, 64), (1 << 31, 64), (1 << 32, 64),
          ((1 << 32) + 5, 64), (1 << 70, 64)]


@pytest.mark.parametrize("given,meant", BOUNDS)
def test_a_bound_on_the_lengths_ends_with_the_table(calls, monkeypatch, given, meant):
    """max_seqlen above what the table holds bounds nothing, also where it passes 32 bits."""
    asked = []
    monkeypatch.setattr(attention, "_fp4_bytes",
                        lambda b, hkv, hq, most, dev: asked.append(most) or 0)
    q = torch.zeros(2, 1, 4, 256, dtype=torch.bfloat16)
    lens, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    rows = [torch.zeros(3, 16, 1, 136, dtype=torch.uint8) for _ in range(2)]
    attention.attn_decode_fp4(q, *rows, lens, table, max_seqlen=given)
    rows = [torch.zeros(3, 16, 1, 256, dtype=torch.bfloat16) for _ in range(2)]
    attention.attn_decode(q, *rows, lens, table, max_seqlen=given)
    attention.attn_decode(q.half(), *(x.half() for x in rows), lens, table, max_seqlen=given)
    rows, scales = [x.to(torch.float8_e4m3fn) for x in rows], [torch.ones(3, 16, 1)] * 2
    attention.attn_decode_fp8(q, *rows, *scales, lens, table, max_seqlen=given)
    at = {"mkv_decode_attention_fp4": 13, "mkv_decode_attention_bf16": 13,
          "mkv_decode_attention_f16": 13, "mkv_decode_attention_fp8": 15}
    assert [name for name, _ in calls] == ["mkv_decode_attention_fp4", "mkv_decode_attention_bf16",
                                           "mkv_decode_attention_f16", "mkv_decode_attention_fp8"]
    for name, args in calls:
        assert args[at[name]] == meant, name
    assert asked[-1] == meant


def test_a_torch_without_the_4_bit_type():
    """Everything but 4-bit pools is there without torch.float4_e2m1fn_x2."""
    code = """
import torch
del torch.float4_e2m1fn_x2
from muserve_amd import kv_cache, scheduler
from muserve_amd.kernels import attention, rope
for dtype in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
    cache = kv_cache.PagedKVCache(4, num_layers=1, kv_heads=1, dtype=dtype, device="cpu",
                                  verbose=False)
    assert cache.dtype == dtype and cache.cache.dtype == dtype
    assert kv_cache._DTYPE_MAP[str(dtype).removeprefix("torch.")] == dtype
try:
    kv_cache.PagedKVCache(4, num_layers=1, kv_heads=1, dtype=torch.uint8, device="cpu")
    raise AssertionError("a pool of uint8")
except ValueError:
    pass
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    assert _DTYPE_MAP["float4_e2m1fn_x2"] == torch.float4_e2m1fn_x2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2])
def test_a_gather_reads_inside_the_pool_and_its_arguments(calls, dtype):
    cache = pool(dtype, layers=3, heads=2)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for layer in (3, -4, 7):
        with pytest.raises(IndexError):
            cache.gather(layer, table, lens)
    for layers in (4, -1):
        with pytest.raises(ValueError, match="layers"):
            cache.gather(None, table, lens, num_layers=layers)
    with pytest.raises(ValueError, match="entry"):
        cache.gather(0, table, lens[:1])
    with pytest.raises(ValueError, match="entry"):
        cache.gather(0, table, lens, starts=lens[:1])
    assert not calls
    k, _ = cache.gather(-1, table, lens, starts=lens)
    assert k.shape == (2, 16, 2, 256)
    assert cache.gather(None, table, lens)[0].shape == (3, 2, 16, 2, 256)
    assert cache.gather(None, table, torch.zeros(5, dtype=torch.int32), num_layers=2)[1].shape[0] == 2
    assert len(calls) == 3
    plane = 2 * 4 * 16 * cache._row_bytes
    assert [args[0] - cache.cache.data_ptr() for _, args in calls] == [2 * plane, 0, 0]


def test_every_query_has_a_length_and_a_table(calls):
    """Over each kind of pool: fewer lengths or rows of the page table than queries are refused."""
    q = torch.zeros(3, 1, 4, 256, dtype=torch.bfloat16)
    lens, table = torch.zeros(3, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.int32)
    wide = torch.zeros(2, 16, 1, 256, dtype=torch.bfloat16)
    codes, scale = wide.to(torch.float8_e4m3fn), torch.ones(2, 16, 1)
    rows = torch.zeros(2, 16, 1, 136, dtype=torch.uint8)
    for fn, x, caches in ((attention.attn_decode, q, (wide, wide)),
                          (attention.attn_decode, q.half(), (wide.half(), wide.half())),
                          (attention.attn_decode_fp8, q, (codes, codes, scale, scale)),
                          (attention.attn_decode_fp4, q, (rows, rows))):
        with pytest.raises(ValueError, match="do not match"):
            fn(x, *caches, lens[:2], table)
        with pytest.raises(ValueError, match="do not match"):
            fn(x, *caches, lens, table[:2])
    assert not calls


def library(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.mkv_last_error().decode()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("append", [False, True])
def test_rows_of_a_rotation_fit_a_grid(dim, append):
    """A grid dimension has fewer than 2^32 threads; dim / 8 of them own a token."""
    row = 2 * dim
    pools = (1, FAKE, FAKE, None, None, 16, FAKE, FAKE) if append else (FAKE,)
    for tokens in ((1 << 35) // dim, (1 << 31) - 1):
        got, text = library("mkv_append_rope" if append else "mkv_qk_norm_rope", FAKE, row, row,
                            FAKE, row, row, *((FAKE, row, row) if append else ()), tokens, 1, 1, dim,
                            0, FAKE, FAKE, 0, 16, 0, 1.0, None, None, 0, 0, 1e-6, FAKE, *pools, None)
        assert got == -3 and "too many rows" in text


@pytest.mark.parametrize("tokens,heads", [(1 << 28, 1), ((1 << 28) - 15, 1), (1 << 27, 2),
                                          (1 << 20, 256)])
def test_rows_of_a_4_bit_append_fit_a_grid(tokens, heads):
    got, text = library("mkv_append_fp4", FAKE, FAKE, 0, 16, FAKE, FAKE, 0, 512, FAKE, tokens, 1,
                        heads, 256, FAKE, None)
    assert got == -3 and "too many rows" in text


@pytest.mark.parametrize("out_len", [1 << 28, (1 << 28) - 15, (1 << 31) - 1])
def test_rows_of_a_4_bit_gather_fit_a_grid(out_len):
    got, text = library("mkv_gather_dequant_fp4", FAKE, FAKE, 0, 4, FAKE, 4, 4, FAKE, None, 1, out_len,
                        None, FAKE, FAKE, 0, 1, 1, 256, FAKE, None)
    assert got == -3 and "out_len" in text


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn, torch.float4_e2m1fn_x2])
@pytest.mark.parametrize("current", [False, True])
def test_launches_on_the_tensors_device(calls, monkeypatch, dtype, current):
    """With another device as the current one, each launch is made with the tensors' as the
    current one: a default stream is the current device's."""
    on, made = [], []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            on.append(self.dev)

        def __exit__(self, *exc):
            on.pop()

    monkeypatch.undo()
    monkeypatch.setattr(_lib, "require_gpu", lambda *tensors: CPU)
    monkeypatch.setattr(_lib, "_device_index", lambda: CPU.index if current else 0)
    monkeypatch.setattr(_lib, "call", lambda name, *args: made.append((name, list(on))))
    monkeypatch.setattr(_lib, "stream_of", lambda dev: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(PagedKVCache, "_gpu", lambda self: self.device)
    for module, kept in ((rope, "_plans"), (attention, "_fp4_plans")):
        monkeypatch.setattr(module, kept, {})
    monkeypatch.setattr(attention, "_errword", lambda dev: _lib.DeviceErrors(CPU))
    monkeypatch.setattr(attention, "_prefill_cus", lambda dev: 256)
    monkeypatch.setattr(attention, "_fp4_bytes", lambda *shape: 0)
    monkeypatch.setattr(attention, "_decode_scratch", lambda *shape: torch.zeros(16))
    monkeypatch.setattr(attention, "_scratch", lambda n, dev: torch.zeros(16))

    cache, slots = pool(dtype), torch.arange(3)
    x = torch.zeros(3, 1, 256, dtype=torch.bfloat16)
    table, lens = torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    cache.append(slots, x, x, layer=0)
    cache.append_rope(slots, x, x, x, 0, torch.arange(3), torch.ones(32))
    cache.gather(0, table, lens)
    cache.copy_pages([1], [2])
    q = torch.zeros(3, 1, 4, 256, dtype=torch.bfloat16)
    if dtype == torch.bfloat16:
        attention.attn_decode(q, *cache.get_kv_by_layer(0), lens, table)
        attention.attn_decode(q, *(torch.zeros(3, 8, 1, 256, dtype=dtype),) * 2, lens, None)
        cu = torch.arange(4, dtype=torch.int32)
        attention.attn_prefill(q[:, 0], x, x, cu, cu, 1, 1)
        attention.attn_prefill_paged(q[:, 0], *cache.get_kv_by_layer(0), cu, lens, table, 1)
    elif dtype == torch.float8_e4m3fn:
        attention.attn_decode_fp8(q, *cache.get_kv_by_layer(0), cache.scales[0, 0],
                                  cache.scales[0, 1], lens, table)
    else:
        attention.attn_decode_fp4(q, *cache.get_kv_by_layer(0), lens, table)
    check = _lib.UniqueCheck(CPU, 16)
    check.run(slots, cache._errors)
    assert len(made) == {torch.bfloat16: 9, torch.float8_e4m3fn: 7, torch.float4_e2m1fn_x2: 6}[dtype]
    for name, entered in made:
        assert entered == ([] if current else [CPU]), name


def test_what_a_tensor_spans():
    x = torch.zeros(4, 3, 8, dtype=torch.bfloat16)
    at = x.data_ptr()
    assert _lib.span(x) == (at, at + 192)
    assert _lib.span(x[1:, ::2, 2:5]) == (at + 52, at + 3 * 48 + 2 * 16 + 10)
    assert _lib.span(x[:0])[1] - _lib.span(x[:0])[0] == 0
    assert _lib.span(x[0, 0, :1].expand(7)) == (at, at + 2)


def test_decode_outputs_that_overlap(calls, monkeypatch):
    monkeypatch.setattr(attention, "_fp4_bytes", lambda *shape: 0)
    flat = torch.zeros(8 * 1024, dtype=torch.bfloat16)
    q = flat[:2048].view(2, 1, 4, 256)
    rows = torch.zeros(3, 16, 1, 136, dtype=torch.uint8)
    lens, table = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    for first in (8, 1024, 2040):
        with pytest.raises(ValueError, match="overlaps"):
            attention.attn_decode_fp4(q, rows, rows, lens, table,
                                      out=flat[first:first + 2048].view(2, 1, 4, 256))
    cache = rows.view(torch.bfloat16).flatten()[8:2056].view(2, 1, 4, 256)
    with pytest.raises(ValueError, match="overlaps"):
        attention.attn_decode_fp4(q, rows, rows, lens, table, out=cache)
    assert not calls
    attention.attn_decode_fp4(q, rows, rows, lens, table, out=q)
    attention.attn_decode_fp4(q, rows, rows, lens, table, out=flat[2048:4096].view(2, 1, 4, 256))
    assert len(calls) == 2
