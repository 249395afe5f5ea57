"""Arguments of the attention layer's operators that are settled before a launch: what reaches
the library, and what does not. The launches themselves are replaced, so no GPU is needed."""
import pytest
import torch

from muserve_amd import _lib
from muserve_amd.kernels import rope
from muserve_amd.kv_cache import PagedKVCache

CPU = torch.device("cpu")


@pytest.fixture
def calls(monkeypatch):
    """The launches that would have been made: (entry point, arguments)."""
    made = []
    monkeypatch.setattr(rope, "_plans", {})  # (what is kept here is of no device)
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
