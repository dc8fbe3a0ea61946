"""CPU: what the microscaled operators' Python side decides before anything is launched."""
import copy
import pickle

import pytest
import torch

from mpq_amd import mx
from mpq_amd.kv_cache import QuantizedKVCache


@pytest.fixture
def on_cpu(monkeypatch):
    """Tensors on the CPU pass for device tensors: nothing is launched here."""
    monkeypatch.setattr(mx, "_on_device", lambda *ts: ts[0].device)


def _cache(**k):
    return QuantizedKVCache(3, 16, 2, 64, device="cpu", **k)


def test_a_cache_keeps_its_tensors_and_shape(on_cpu):
    """The calls hold addresses: a tensor or a size that were replaced would be memory that is gone, or reads past it."""
    c = _cache(fmt="mxfp4")
    before = {n: getattr(c, n) for n in c._FIXED}
    for name in sorted(c._FIXED):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(c, name, torch.zeros(1))
        with pytest.raises(AttributeError, match="fixed"):
            delattr(c, name)
    assert all(getattr(c, n) is v for n, v in before.items())
    c.note = 1  # a user's own attribute
    c.note = 2
    del c.note


@pytest.mark.parametrize("way", [copy.copy, copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))])
def test_a_copied_cache_addresses_its_own_tensors(on_cpu, way):
    c = _cache(dtype=torch.float16)
    d = way(c)
    tensors = (d.k_codes, d.k_scales, d.v_codes, d.v_scales)
    assert d._call == (*c._call[:5], *(t.data_ptr() for t in tensors))
    assert (d.fmt, d.dtype, d.num_pages, d.heads, d.page_size, d.head_dim) == ("mxfp8", torch.float16, 3, 2, 16, 64)
    assert (d.k_codes is c.k_codes) == (way is copy.copy)


def test_a_quantised_tensor_keeps_what_was_checked(on_cpu):
    """The kernels go by the sizes that the constructor checked against the tensors."""
    t = mx.MXTensor(torch.zeros(6, 128, dtype=torch.uint8), torch.ones(6, 8, dtype=torch.uint8), 200, lead=(2, 3))
    for name, value in (("codes", t.codes[:2]), ("scales", t.scales[:2]), ("rows", 7), ("cols", 900), ("fmt", "mxfp8"),
                        ("lead", (6,)), ("device", None), ("shape", (6, 200))):
        with pytest.raises(AttributeError):
            setattr(t, name, value)
        with pytest.raises(AttributeError):
            delattr(t, name)
    for u in (t, copy.copy(t), copy.deepcopy(t), pickle.loads(pickle.dumps(t))):
        assert (u.shape, u.rows, u.cols, u.lead, u.fmt) == ((2, 3, 200), 6, 200, (2, 3), "mxfp4")
        assert torch.equal(u.codes, t.codes) and torch.equal(u.scales, t.scales) and u.device == t.device


def test_a_backward_pass_raises():
    """Results hold no gradient: where one would be recorded, its backward pass says so instead of leaving it out."""
    x, bias = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    for inputs in ((x,), (None, bias), (x, bias)):
        out = torch.zeros(3)
        got = mx._no_gradient("op", out, *inputs)
        assert got.requires_grad and got.data_ptr() == out.data_ptr()
        with pytest.raises(RuntimeError, match="op has no gradient"):
            (got * 2 + x).sum().backward()
    out = torch.zeros(3)
    assert mx._no_gradient("op", out, x.detach(), None) is out and mx._no_gradient("op", out, None) is out
    with torch.no_grad():
        assert mx._no_gradient("op", out, x) is out and not out.requires_grad
