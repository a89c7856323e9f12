"""CPU: calls that copy several inputs (tensors that are not contiguous) hand the library copies that all live until the call is made."""
import ctypes as C
import types

import pytest
import torch

import util
from justgoal_b200 import main as M


class Recorder:
    """Stands for the library: reads what each pointer of a call points to, while the call is made."""

    def __init__(self, sizes):
        self.sizes, self.seen = sizes, []

    def __call__(self, handle, *args):
        self.seen = [C.string_at(a.value, n) for a, n in zip(args, self.sizes) if n]
        return 0


def _layer(monkeypatch, name, sizes):
    layer = M.MoELayer.__new__(M.MoELayer)
    layer.shape, layer._h = util.I.TINY_RENORM, None
    monkeypatch.setattr(M.MoELayer, "__del__", lambda self: None, raising=False)
    monkeypatch.setattr(M.MoELayer, "ep_row_bytes", lambda self: 64)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=0))
    rec = Recorder(sizes)
    monkeypatch.setattr(M._lib, "lib", types.SimpleNamespace(**{"b200moe_" + name: rec}))
    return layer, rec


def _columns(t):
    """The same values, stored by columns."""
    out = t.t().contiguous().t()
    assert not out.is_contiguous()
    return out


def _bytes(t):
    return t.contiguous().view(torch.uint8).numpy().tobytes()


@pytest.mark.parametrize("T", [2, 33, 400])
def test_ep_pack(monkeypatch, T):
    g = torch.Generator().manual_seed(T)
    H, K = 384, 4
    ins = [torch.randint(0, 100, (T, H), generator=g, dtype=torch.uint8), torch.randn(H // 128, T, generator=g), torch.randint(0, 32, (T, K), generator=g, dtype=torch.int32),
           torch.rand(T, K, generator=g)]
    send = torch.arange(2 * T)[::2]
    layer, rec = _layer(monkeypatch, "ep_pack", [t.nbytes for t in (*ins, send)])
    layer.ep_pack(*[_columns(t) for t in ins], send)
    assert rec.seen == [_bytes(t) for t in (*ins, send)]


@pytest.mark.parametrize("T", [2, 33, 400])
def test_ep_combine(monkeypatch, T):
    g = torch.Generator().manual_seed(T)
    rows, row_of = torch.randn(T, 384, generator=g).half(), torch.randint(0, T, (2, T), generator=g, dtype=torch.int32)
    layer, rec = _layer(monkeypatch, "ep_combine", [rows.nbytes, row_of.nbytes])
    layer.ep_combine(_columns(rows), _columns(row_of), T)
    assert rec.seen == [_bytes(rows), _bytes(row_of)]
