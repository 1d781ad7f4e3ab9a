"""The axes of rotary frequencies, and what norm_rope_heads and its C entry refuse before any device is touched."""
import pytest
import torch

from heimdall_b200 import _lib, norm_rope_heads, rope_axes


def test_axes_are_dealt_in_turn():
    assert rope_axes((3, 2, 2)) == [0, 1, 2, 0, 1, 2, 0]
    assert rope_axes((4, 1, 0)) == [0, 1, 0, 0, 0]
    assert rope_axes((11, 11, 10)).count(1) == 11 and len(rope_axes((11, 11, 10))) == 32
    assert rope_axes((8,)) == [0] * 8
    for bad in ((1, 3, 0), (2, 3, 3), (-1, 2), (), (1, 1, 1, 1, 1)):
        with pytest.raises(ValueError):
            rope_axes(bad)


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 1, 1, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        norm_rope_heads(x, x, torch.zeros(256), torch.zeros(256), torch.zeros(1, 1, dtype=torch.int32), None, gated=False)


def _call(**kw):
    a = dict(qg=16, kl=16, w=16, freqs=8, axes=bytes(8), n_axes=1, pos=16, eps=1e-6, B=1, T=1, H=1, G=1, D=256, dtype=1, q=16, k=16, qr=16,
             kr=16, qs=256)
    a.update(kw)
    _lib.call("bf_norm_rope", a["qg"], 0, 0, a["qs"], a["kl"], 0, 0, 256, a["w"], a["w"], 16, a["freqs"], a["axes"], a["n_axes"], a["pos"], 0,
              a["eps"], a["B"], a["T"], a["H"], a["G"], a["D"], a["dtype"], a["q"], a["k"], a["qr"], a["kr"], 0)


@pytest.mark.parametrize("code,kw", [(1, {"qg": 0}), (1, {"qr": 0}), (1, {"q": 0}), (1, {"pos": 0}), (1, {"axes": None}), (1, {"B": -1}), (1, {"H": 0}),
                                     (1, {"freqs": 12}), (1, {"freqs": 136}), (1, {"n_axes": 5}), (1, {"n_axes": 0}), (1, {"eps": -1.0}),
                                     (1, {"eps": float("nan")}), (1, {"axes": bytes([0, 0, 0, 1, 0, 0, 0, 0])}), (2, {"D": 128}),
                                     (2, {"dtype": 0}), (3, {"qg": 8}), (3, {"kr": 24}), (3, {"qs": 260})])
def test_c_entry_refuses(code, kw):
    with pytest.raises(_lib.BifrostError) as e:
        _call(**kw)
    assert e.value.code == code


def test_c_entry_takes_no_tokens():
    _call(T=0, qg=0, kl=0)
    _call(B=0)


@pytest.mark.parametrize("kw", [{"w": 18}, {"pos": 18}, {"pos": 20, "pos64": 1}])
def test_c_entry_refuses_what_is_not_on_its_types_boundary(kw):
    a = dict(w=20, pos=20, pos64=0)
    a.update(kw)
    with pytest.raises(_lib.BifrostError) as e:
        _lib.call("bf_norm_rope", 16, 0, 0, 256, 16, 0, 0, 256, a["w"], a["w"], 20, 8, bytes(8), 1, a["pos"], a["pos64"], 1e-6, 1, 1, 1, 1, 256, 1,
                  16, 16, 16, 16, 0)
    assert e.value.code == 3
