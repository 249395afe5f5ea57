"""The 4-bit pool's and the rotation's entry points: refused arguments come back as status
codes without touching a GPU; the pool's arithmetic on the host."""
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels.rope import qk_norm_rope
from muserve_amd.kv_cache import PagedKVCache

FAKE = 1 << 20  # an aligned non-null address; argument checks fail before any use


def rc(name, *args):
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.mkv_last_error().decode()


def append(**change):
    a = dict(kp=FAKE, vp=FAKE, stride=0, slots=16, k=FAKE, v=FAKE, layer=0, tok=512, map=FAKE,
             tokens=1, layers=1, heads=1, dim=256, err=FAKE, stream=None)
    a.update(change)
    return rc("mkv_append_fp4", *a.values())


@pytest.mark.parametrize("change,code,text", [
    (dict(dim=128), -3, "head_dim 128"), (dict(heads=0), -1, "bad size"),
    (dict(tokens=-1), -1, "bad size"), (dict(kp=None), -1, "null pointer"),
    (dict(k=FAKE + 8), -2, "misaligned"), (dict(tok=520), -2, "misaligned"),
    (dict(tokens=1 << 31), -3, "too many rows"), (dict(tokens=1 << 30, heads=4), -3, "too many"),
    (dict(layers=40000), -3, "too many rows")])
def test_append_refusals(change, code, text):
    got, msg = append(**change)
    assert got == code and text in msg


def test_empty_appends():
    assert append(tokens=0, kp=None)[0] == 0 and append(layers=0, k=None)[0] == 0


def gather(**change):
    a = dict(kp=FAKE, vp=FAKE, stride=0, pages=4, table=FAKE, tstride=4, width=4, lens=FAKE,
             starts=None, batch=1, out_len=16, offs=None, k=FAKE, v=FAKE, layer=0, layers=1, heads=1,
             dim=256, err=FAKE, stream=None)
    a.update(change)
    return rc("mkv_gather_dequant_fp4", *a.values())


@pytest.mark.parametrize("change,code", [
    (dict(dim=64), -3), (dict(heads=0), -1), (dict(heads=2000), -3), (dict(batch=-1), -1),
    (dict(batch=70000), -3), (dict(out_len=1 << 31), -3), (dict(lens=None), -1),
    (dict(k=FAKE + 8), -2), (dict(stride=8), -2), (dict(offs=FAKE, layer=-16), -1),
    (dict(layers=40000), -3)])
def test_gather_refusals(change, code):
    assert gather(**change)[0] == code


def decode(**change):
    a = dict(q=FAKE, k=FAKE, v=FAKE, pages=4, shared=0, hkv=1, hq=4, dim=256, table=FAKE, tstride=4,
             width=4, lens=FAKE, batch=1, most=1 << 20, scale=0.0625, out=FAKE, ws=FAKE, bytes=1 << 40,
             err=FAKE, stream=None)
    a.update(change)
    return rc("mkv_decode_attention_fp4", *a.values())


@pytest.mark.parametrize("change,code", [
    (dict(dim=128), -3), (dict(hq=9), -3), (dict(hq=5, hkv=2), -3), (dict(hq=2, hkv=4), -3),
    (dict(batch=4097), -3), (dict(batch=4096, hkv=2, hq=2), -3), (dict(most=(1 << 24) + 1), -3),
    (dict(batch=4096, most=1 << 24), -3), (dict(pages=0), -1), (dict(shared=-1), -1),
    (dict(tstride=3), -1), (dict(q=None), -1), (dict(table=None), -1), (dict(k=FAKE + 8), -2),
    (dict(bytes=100), -1), (dict(ws=None), -1), (dict(ws=FAKE + 8), -1), (dict(most=-1), -1)])
def test_decode_refusals(change, code):
    got, msg = decode(**change)
    assert got == code and msg


def test_empty_decode_and_workspaces():
    assert decode(batch=0, q=None, ws=None)[0] == 0
    size = _lib.load().mkv_decode_attention_fp4_workspace_bytes
    long = 1 << 20
    assert size(1, 1, 4, long) > 0 and size(4096, 1, 8, long) > size(1, 1, 8, long)
    assert size(1, 1, 4, 512) == 0 < size(4096, 1, 4, 512)
    for bad in ((1, 1, 9, long), (4097, 1, 1, 9), (1, 2, 3, 9), (-1, 1, 1, 9), (1, 0, 1, 9),
                (1, 1, 1, -1)):
        assert size(*bad) == -1


def rope(fn="mkv_qk_norm_rope", **change):
    a = dict(q=FAKE, qt=2048, qh=512, k=FAKE, kt=512, kh=512)
    if fn == "mkv_append_rope":
        a.update(v=FAKE, vt=512, vh=512)
    a.update(tokens=1, hq=4, hk=1, dim=256, fp16=0, pos=FAKE, freq=FAKE, f64=0, rot=64, pairs=0,
             scale=1.0, qw=FAKE, kw=FAKE, kind=1, centred=0, eps=1e-6, qo=FAKE)
    if fn == "mkv_append_rope":
        a.update(pool=1, kp=FAKE, vp=FAKE, ks=None, vs=None, slots=16, map=FAKE, err=FAKE)
    else:
        a.update(ko=FAKE)
    a.update(stream=None)
    a.update(change)
    return rc(fn, *a.values())


@pytest.mark.parametrize("fn", ["mkv_qk_norm_rope", "mkv_append_rope"])
@pytest.mark.parametrize("change,code", [
    (dict(dim=96), -3), (dict(dim=512), -3), (dict(rot=0), -3), (dict(rot=40), -3),
    (dict(rot=272), -3), (dict(tokens=-1), -1), (dict(tokens=1 << 31), -3), (dict(hq=70000), -3),
    (dict(kind=4), -1), (dict(q=None), -1), (dict(qo=None), -1), (dict(k=None), -1),
    (dict(pos=None), -1), (dict(freq=None), -1), (dict(q=FAKE + 8), -2), (dict(qt=2040), -2),
    (dict(kh=8), -2), (dict(qw=FAKE + 2), -2), (dict(freq=FAKE + 4, f64=1), -2)])
def test_rope_refusals(fn, change, code):
    got, msg = rope(fn, **change)
    assert got == code and msg


@pytest.mark.parametrize("change,code", [
    (dict(pool=0), -1), (dict(pool=4), -1), (dict(pool=3, fp16=1), -3), (dict(pool=2, dim=128), -3),
    (dict(pool=2), -1), (dict(hk=0), -1), (dict(v=None), -1), (dict(kp=None), -1),
    (dict(map=None), -1), (dict(err=None), -1), (dict(vt=8), -2), (dict(kp=FAKE + 8), -2)])
def test_append_rope_refusals(change, code):
    got, msg = rope("mkv_append_rope", **change)
    assert got == code and msg


def test_empty_ropes():
    assert rope(tokens=0, q=None)[0] == 0 and rope(hq=0, hk=0, q=None)[0] == 0
    assert rope("mkv_append_rope", tokens=0, kp=None)[0] == 0


def test_the_pool_on_the_host():
    cache = PagedKVCache(10, num_layers=3, kv_heads=2, dtype=torch.float4_e2m1fn_x2, device="cpu",
                         verbose=False)
    assert cache.cache.shape == (3, 2, 10, 16, 2, 136) and cache.cache.dtype == torch.uint8
    assert cache.scales is None and cache.dtype == torch.float4_e2m1fn_x2
    assert cache.get_kv_by_layer(1)[1].shape == (10, 16, 2, 136)
    with pytest.raises(ValueError, match="256"):
        PagedKVCache(4, num_layers=1, kv_heads=1, head_dim=128, dtype=torch.float4_e2m1fn_x2,
                     device="cpu", verbose=False)
    with pytest.raises(RuntimeError, match="need a ROCm GPU"):
        cache.append(torch.zeros(1, dtype=torch.int64), torch.zeros(1, 2, 256), torch.zeros(1, 2, 256),
                     layer=0)
    with pytest.raises(RuntimeError, match="need a ROCm GPU"):
        cache.append_rope(torch.zeros(1, dtype=torch.int64), None, None, None, 0, None, None)


def test_pages_of_a_4_bit_pool(monkeypatch):
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda d: (10 ** 9, 10 ** 9))
    pages = PagedKVCache._estimate_pages("cuda:0", 2, torch.float4_e2m1fn_x2, 5, 256)
    assert pages == 900_000_000 // (5 * 2 * 16 * 2 * 136)


def test_no_fallback_off_the_gpu():
    x = torch.zeros(1, 1, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="ROCm GPU only"):
        qk_norm_rope(x, x, torch.zeros(1, dtype=torch.int64), torch.ones(32))
