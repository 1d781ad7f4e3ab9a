"""What Adapters and its C entries refuse before any device is touched, and the workspace they ask for."""
import pytest
import torch

from heimdall_b200 import Adapters, _lib

bf = torch.bfloat16


def _pair(r=8, i=64, o=32, dtype=bf):
    return torch.zeros(r, i, dtype=dtype), torch.zeros(o, r, dtype=dtype)


def test_adapters_are_refused():
    a, b = _pair()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        Adapters([a], [b])
    for bad in (([], []), ([a], [b, b]), ([a], [_pair(4)[1]]), ([a, _pair(8, 72)[0]], [b, b]), ([a, _pair()[0].half()], [b, b]),
                ([a[0]], [b])):
        with pytest.raises(ValueError):
            Adapters(*bad, device="cuda")
    with pytest.raises(ValueError, match="scale"):
        Adapters([a], [b], [1.0, 2.0], device="cuda")
    for bad in (_pair(129), _pair(0), _pair(8, 60), _pair(8, 64, 20), _pair(dtype=torch.float32)):
        with pytest.raises(NotImplementedError):
            Adapters([bad[0]], [bad[1]], device="cuda")


def _call(**kw):
    a = dict(x=16, xs=64, ids=16, T=4, d_in=64, d_out=32, A=16, B=16, row=16, scale=16, n=2, rmax=16, y=16, ys=32, out=16, os=32, dtype=1, ws=16,
             nws=1 << 20)
    a.update(kw)
    _lib.call("bf_adapter_add", *a.values(), 0)


@pytest.mark.parametrize("code,kw", [(1, {"x": 0}), (1, {"ids": 0}), (1, {"out": 0}), (1, {"T": -1}), (1, {"n": 0}), (1, {"d_in": 0}), (2, {"d_in": 60}),
                                     (2, {"d_out": 36}), (2, {"rmax": 24}), (2, {"rmax": 144}), (2, {"n": 4097}), (2, {"dtype": 0}),
                                     (2, {"T": 1 << 29}), (3, {"x": 8}), (3, {"ys": 36}), (3, {"ws": 8}), (4, {"ws": 0}), (4, {"nws": 100})])
def test_c_entry_refuses(code, kw):
    with pytest.raises(_lib.BifrostError) as e:
        _call(**kw)
    assert e.value.code == code


def test_workspace_and_no_tokens():
    _call(T=0, x=0, ws=0)
    size = lambda *a: _lib.size("bf_adapter_workspace", *a)
    assert size(0, 2, 64, 16) == size(4, 4097, 64, 16) == size(4, 2, 64, 144) == 0
    assert size(64, 61, 5120, 32) >= 5 * 64 * 32 * 4
    assert size(8192, 4, 5120, 64) >= 8192 * 64 * 4 + 8192 * 4


@pytest.mark.parametrize("adapters", [{}, {"q": None}])
def test_adapter_ids_are_checked_with_and_without_adapters(adapters):
    from heimdall_b200 import BifrostAttention
    layer = BifrostAttention.__new__(BifrostAttention)
    layer.adapters = adapters
    x = torch.zeros(3, 90, 8)
    for bad in (torch.zeros(2), torch.zeros(2, dtype=torch.int64), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3), torch.zeros(3, 90, dtype=torch.bool)):
        with pytest.raises(ValueError, match="adapter_ids"):
            layer._ids(x, bad)
    ids = torch.tensor([2 ** 40, -1, 2])
    got = layer._ids(x, ids)
    assert layer._ids(x, None) is None and (got is None) == (not adapters)
    if adapters:
        assert got.dtype == torch.int32 and got.is_contiguous() and got[:, 7].tolist() == [2 ** 31 - 1, -1, 2]
