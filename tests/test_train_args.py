"""CPU: the training operators' C ABI exports what include/b200moe_train.h declares, and refuses bad arguments before it touches a
device; the Python entry points refuse bad tensors."""
import ctypes as C
import os
import re

import pytest
import torch

import util
from justgoal_b200 import _lib

lib = _lib.lib
P = C.c_void_p(1 << 20)        # an aligned address that no refused call looks at
ODD = C.c_void_p((1 << 20) + 4)


def test_library_exports_every_declared_symbol():
    src = open(os.path.join(util.ROOT, "include", "b200moe_train.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    names = set(re.findall(r"\b(b200moe_[a-z_0-9]+)\s*\(", src))
    assert len(names) == 9
    loaded = C.CDLL(_lib.LIB_PATH)
    for name in names:
        assert hasattr(loaded, name) and getattr(lib, name).argtypes is not None, name


def test_sort_refuses():
    n = C.c_size_t(77)
    assert lib.b200moe_sort_workspace_bytes(4, 8, 32, None) == -1
    for T, K, El in ((-1, 8, 32), (4, 0, 32), (4, 9, 32), (4, 8, 0), (4, 8, 513), (1 << 28, 8, 32)):
        assert lib.b200moe_sort_workspace_bytes(T, K, El, C.byref(n)) == -1
        assert lib.b200moe_sort_tokens(P, T, K, El, 0, 16, 100, P, P, P, None, 0, None) == -1
    assert lib.b200moe_sort_workspace_bytes(3, 8, 32, C.byref(n)) == 0 and n.value == 0
    for align in (0, -16, 3, 24, 256):
        assert lib.b200moe_sort_tokens(P, 4, 8, 32, 0, align, 100, P, P, P, None, 0, None) == -1
    assert lib.b200moe_sort_tokens(P, 4, 8, 32, 0, 16, -1, P, P, P, None, 0, None) == -1
    for args in ((None, P, P, P), (P, None, P, P), (P, P, None, P), (P, P, P, None)):
        assert lib.b200moe_sort_tokens(args[0], 4, 8, 32, 0, 16, 100, args[1], args[2], args[3], None, 0, None) == -1
    assert lib.b200moe_sort_workspace_bytes(9000, 8, 32, C.byref(n)) == 0 and n.value > 0
    assert lib.b200moe_sort_tokens(P, 9000, 8, 32, 0, 16, 100, P, P, P, None, n.value, None) == -2
    assert lib.b200moe_sort_tokens(P, 9000, 8, 32, 0, 16, 100, P, P, P, P, n.value - 1, None) == -2


def _row_calls(type=0, T=4, K=8, El=32, H=128, R=100, x=P, row0=P, row_pair=P, pair_row=P, rows=P, w=P, scale=P, out=P):
    """The answers of permute, restore_1x128, combine and combine_backward to one set of arguments."""
    return [lib.b200moe_permute(x, type, row0, row_pair, pair_row, T, K, El, H, R, rows, None),
            lib.b200moe_restore_1x128(x, scale, type, row0, row_pair, pair_row, T, K, El, H, R, rows, None),
            lib.b200moe_combine(rows, type, w, pair_row, T, K, H, R, out, None),
            lib.b200moe_combine_backward(out, rows, type, w, row0, row_pair, pair_row, T, K, El, H, R, x, P, None)]


@pytest.mark.parametrize("bad", [dict(type=3), dict(type=-1), dict(T=-1), dict(K=0), dict(K=9), dict(H=0), dict(H=100), dict(H=-128), dict(R=-1),
                                 dict(H=(1 << 20) + 128), dict(R=(1 << 30) + 1),
                                 dict(T=1 << 28), dict(pair_row=None), dict(rows=None), dict(rows=ODD)])
def test_row_operators_refuse(bad):
    assert _row_calls(**bad) == [-1] * 4


def test_row_operators_refuse_what_only_some_take():
    for bad in (dict(El=0), dict(El=513), dict(row0=None), dict(row_pair=None), dict(x=None), dict(x=ODD)):
        got = _row_calls(**{**bad, "out": None})          # (out None: the combine stays out of it)
        assert got == [-1] * 4, bad
    assert lib.b200moe_restore_1x128(P, None, 0, P, P, P, 4, 8, 32, 128, 100, P, None) == -1
    assert lib.b200moe_restore_1x128(P, P, 0, None, None, None, 4, 8, 32, 100, 0, P, None) == -1
    assert lib.b200moe_restore_1x128(P, P, 0, P, None, None, 4, 8, 32, 128, 100, P, None) == -1          # some tables, not all
    assert lib.b200moe_combine(P, 0, None, P, 4, 8, 128, 100, None, None) == -1
    assert lib.b200moe_combine_backward(P, P, 0, None, P, P, P, 4, 8, 32, 128, 100, P, P, None) == -1
    assert lib.b200moe_combine_backward(P, P, 0, P, P, P, P, 4, 8, 32, 128, 100, P, None, None) == -1


def test_nothing_to_do_needs_no_device():
    assert lib.b200moe_permute(None, 0, None, None, None, 0, 8, 32, 128, 0, None, None) == 0
    assert lib.b200moe_restore_1x128(None, None, 0, None, None, None, 0, 8, 32, 128, 0, None, None) == 0
    assert lib.b200moe_combine(None, 0, None, None, 0, 8, 128, 0, None, None) == 0
    assert lib.b200moe_combine_backward(None, None, 0, None, None, None, None, 0, 8, 32, 128, 0, None, None, None) == 0
    assert lib.b200moe_swiglu_save(None, 0, None, 0, 128, None, None, None, None) == 0
    assert lib.b200moe_swiglu_backward(None, None, None, 0, None, 0, 128, None, None, None) == 0
    assert lib.b200moe_route_backward(None, None, None, None, 0, 64, 8, 1.0, 0, None, None) == 0


def test_swiglu_refuses():
    good = dict(x=P, type=0, used=None, R=4, I=128, act=P, q=P, scale=P)

    def save(**kw):
        a = {**good, **kw}
        return lib.b200moe_swiglu_save(a["x"], a["type"], a["used"], a["R"], a["I"], a["act"], a["q"], a["scale"], None)

    def grad(**kw):
        a = {**good, **kw}
        return lib.b200moe_swiglu_backward(a["q"], a["scale"], a["x"], a["type"], a["used"], a["R"], a["I"], a["gx"] if "gx" in kw else P, a["act"], None)

    for bad in (dict(type=3), dict(R=-1), dict(R=(1 << 30) + 1), dict(I=0), dict(I=100), dict(I=(1 << 20) + 128), dict(x=None), dict(x=ODD), dict(q=None), dict(q=ODD),
                dict(scale=None), dict(act=ODD)):
        assert save(**bad) == -1 and grad(**bad) == -1, bad
    assert save(act=None) == -1 and grad(gx=None) == -1 and grad(gx=ODD) == -1


def test_route_backward_refuses():
    def call(logits=P, idx=P, d=P, T=4, E=64, K=8, mode=0, out=P):
        return lib.b200moe_route_backward(logits, None, idx, d, T, E, K, 2.5, mode, out, None)

    for bad in (dict(T=-1), dict(E=0), dict(E=40), dict(E=544), dict(K=0), dict(K=9), dict(mode=6), dict(mode=-1), dict(mode=4), dict(logits=None),
                dict(idx=None), dict(d=None), dict(out=None), dict(logits=ODD), dict(out=ODD)):
        assert call(**bad) == -1, bad


def test_python_entry_points_refuse_host_tensors_and_wrong_types():
    import justgoal_b200 as jg
    idx = torch.zeros(4, 8, dtype=torch.int32)
    order = jg.TokenOrder(torch.zeros(33, dtype=torch.int32), torch.zeros(100, dtype=torch.int32), idx)
    x, w = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(4, 8)
    rows, q = torch.zeros(100, 256, dtype=torch.bfloat16), torch.zeros(4, 256).to(torch.float8_e4m3fn)
    for call in (lambda: jg.sort_tokens(idx, 32), lambda: jg.permute(x, order), lambda: jg.permute_backward(rows, order), lambda: jg.combine(rows, w, order),
                 lambda: jg.combine_backward(x, rows, w, order), lambda: jg.restore_1x128(q, torch.zeros(2, 4)), lambda: jg.swiglu_save(rows),
                 lambda: jg.swiglu_backward(q, torch.zeros(2, 4), x), lambda: jg.route_backward(torch.zeros(4, 64), None, idx, w, 1.0)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()
    for call in (lambda: jg.sort_tokens(idx.long(), 32), lambda: jg.sort_tokens(idx[0], 32), lambda: jg.permute(x.double(), order),
                 lambda: jg.permute(x[0], order), lambda: jg.combine(rows.int(), w, order), lambda: jg.swiglu_save(rows.to(torch.int8))):
        with pytest.raises(ValueError):
            call()


def test_sort_workspace_of_a_size_is_enough_for_smaller_ones():
    """Never falls with the pairs or the local experts: the CTAs of a call do, where slices get longer (303104, 606208, ... pairs on 148 SMs)."""
    def size(T, K=8, El=256):
        n = C.c_size_t()
        assert lib.b200moe_sort_workspace_bytes(T, K, El, C.byref(n)) == 0
        return n.value

    steps = [257, 258, 384, 385, 1000, 14107, 37887, 37888, 37889, 40000, 75775, 75776, 75777, 113664, 113665, 1 << 20, 1 << 26, 1 << 27]
    sizes = [size(T) for T in steps]
    assert sizes == sorted(sizes) and sizes[0] > 0
    for T in (256, 5000, 37889):
        by_experts = [size(T, El=El) for El in (1, 4, 5, 32, 255, 256, 512)]
        assert by_experts == sorted(by_experts)
    pairs = [size(T, K=1) for T in range(2000, 320000, 333)]
    assert pairs == sorted(pairs)


@pytest.mark.parametrize("tables", [((2, 33), (100,), (4, 8)), ((33,), (100, 1), (4, 8)), ((33,), (100,), (32,)), ((33,), (100,), (4, 8, 1)), ((), (100,), (4, 8)),
                                    ((33,), (), (4, 8)), ((0,), (100,), (4, 8)), ((1,), (100,), (4, 8)), ((33,), (100,), (4, 9)), ((33,), (100,), (4, 0)), ((514,), (100,), (4, 8))])
def test_orders_of_other_forms_are_refused(tables):
    """Tables of another number of dimensions, of no or too many experts or picks (the check itself, which takes the device's number: -1 is the host)."""
    from justgoal_b200.train import _order
    make = lambda shapes, dtype=torch.int32: [torch.zeros(s, dtype=dtype) for s in shapes]   # noqa: E731
    assert _order(make(((33,), (100,), (4, 8))), -1)[4:] == (4, 8, 32, 100)
    with pytest.raises(ValueError, match="an order"):
        _order(make(tables), -1)
    with pytest.raises(ValueError, match="an order is int32"):
        _order(make(((33,), (100,), (4, 8)), torch.int64), -1)
    with pytest.raises(ValueError, match="an order is int32"):
        _order(make(((33,), (100,), (4, 8))), 0)
