"""Rotary positions: the tables' frequencies and the argument checks, which need no GPU."""

import ctypes
import math
from types import SimpleNamespace

import pytest
import torch

import _capi
import rotary as ro


def frequencies(r, base=10000.0, scaling=None, factor=1.0, original=None, fast=32.0, slow=1.0):
    return ro._frequencies(r, base, scaling, factor, original, fast, slow)


def close(a, b):
    # powers and products of a few roundings each
    assert len(a) == len(b) and all(abs(x - y) <= 2.0 ** -48 * abs(y) for x, y in zip(a, b))


@pytest.mark.parametrize("r", [2, 64, 80, 128, 256])
def test_frequencies(r):
    plain = [math.exp(-2 * j / r * math.log(10000.0)) for j in range(r // 2)]
    f, m = frequencies(r)
    assert m == 1.0
    close(f, plain)
    f, m = frequencies(r, scaling="linear", factor=8.0)
    assert m == 1.0
    close(f, [x / 8 for x in plain])
    if r > 2:
        f, m = frequencies(r, scaling="ntk", factor=8.0)
        assert m == 1.0 and f[0] == 1.0
        close(f[-1:], [plain[-1] / 8])                  # the last pair as linear scaling has it
        close(f, [x * 8.0 ** (-2 * j / (r - 2)) for j, x in enumerate(plain)])


def test_scaled_between_two_turn_counts():
    r, original, factor = 128, 32768, 4.0
    f, m = frequencies(r, scaling="yarn", factor=factor, original=original)
    plain, _ = frequencies(r)
    assert abs(m - (0.1 * math.log(4.0) + 1)) < 1e-15
    for x, p in zip(f, plain):
        turns = original * p / (2 * math.pi)
        assert p / factor * (1 - 1e-15) <= x <= p * (1 + 1e-15)
        if turns > 33 * 1.16:        # a pair past the border: neighbours differ by 10000^(1/64) = 1.155
            assert x == p
        if turns < 1 / 1.16:
            assert abs(x - p / factor) <= 1e-15 * x
    assert any(p / factor < x < p for x, p in zip(f, plain))


def test_given_frequencies_keep_64_bits(monkeypatch):
    """Numbers are not taken through 32 bits, which would move the angle of position 2^20 by 2^-5."""
    monkeypatch.setattr(ro.Rotary, "__post_init__", lambda self: None)
    f = [0.1, 1.0, 1 / 3]
    for given in (f, tuple(f), torch.tensor(f, dtype=torch.float64)):
        assert ro.Rotary.from_frequencies(given).turns.tolist() == [x / (2 * math.pi) for x in f]
    for half in (torch.float32, torch.bfloat16):        # a tensor's values as they are
        t = torch.tensor(f, dtype=half)
        assert ro.Rotary.from_frequencies(t).turns.tolist() == [x / (2 * math.pi) for x in t.tolist()]


def test_bad_tables_are_refused():
    for kw in (dict(r=3), dict(r=0), dict(r=64, base=0.0), dict(r=64, base=math.inf), dict(r=64, scaling="other"),
               dict(r=64, scaling="linear", factor=0.0), dict(r=64, factor=2.0), dict(r=2, scaling="ntk", factor=2.0),
               dict(r=64, scaling="yarn", factor=2.0), dict(r=64, scaling="yarn", factor=0.5, original=100),
               dict(r=64, scaling="yarn", factor=2.0, original=100, fast=1.0, slow=2.0)):
        with pytest.raises(AssertionError):
            frequencies(**kw)
    for turns in (torch.zeros(4, dtype=torch.float64), torch.zeros(4), torch.zeros(0, dtype=torch.float64)):
        with pytest.raises(AssertionError):
            ro.Rotary(turns)                            # host tensors, 32 bits, no pair


def table(r=64):
    return SimpleNamespace(_call=(None, -1, r))


def no_launch(monkeypatch, calls=None):
    monkeypatch.setattr(ro, "_launch", lambda *a: calls.append(a) if calls is not None else None)


def test_refused_arguments(monkeypatch):
    no_launch(monkeypatch)
    bf = torch.bfloat16
    q, k, pos = torch.zeros(5, 4, 64, dtype=bf), torch.zeros(5, 2, 64, dtype=bf), torch.zeros(5, dtype=torch.int32)
    ro.rotary(table(), pos, q, k)
    for bad in (lambda: ro.rotary(table(), pos, q.float()), lambda: ro.rotary(table(), pos, q, k.half()),
                lambda: ro.rotary(table(), pos.long(), q), lambda: ro.rotary(table(), pos[:4], q),
                lambda: ro.rotary(table(), pos.repeat(2)[::2], q), lambda: ro.rotary(table(), pos.view(1, 5), q),
                lambda: ro.rotary(table(), pos, q, k[:4]), lambda: ro.rotary(table(), pos, q, k.view(1, 2, 5, 64)),
                lambda: ro.rotary(table(128), pos, q), lambda: ro.rotary(table(), pos, q[:, :0]),
                lambda: ro.rotary(table(), pos, q[..., :48]), lambda: ro.rotary(table(), pos, q[0]),
                lambda: ro.rotary(table(), pos, q, out=torch.zeros(5, 4, 64)),
                lambda: ro.rotary(table(), pos, q, k, out=torch.zeros_like(q)),
                lambda: ro.rotary(table(), pos, q, out=torch._neg_view(torch.zeros_like(q))),
                lambda: ro.rotary(table(), pos, q, out=torch.zeros(5, 1, 64, dtype=bf).expand(5, 4, 64)),
                lambda: ro.rotary(table(), pos, q, out=torch.zeros(5, 4, 128, dtype=bf)[..., ::2]),
                lambda: ro.rotary(table(), pos, q, out=torch.zeros(5, 4, 64, dtype=bf, requires_grad=True)),
                lambda: ro.rotary(table(), pos, q.clone().requires_grad_(), out=q)):
        with pytest.raises(AssertionError):
            bad()


def test_outputs_over_inputs(monkeypatch):
    """In place is one element on itself; heads of one projection may be turned where they are; anything
    else that overlaps would be read after it is written."""
    calls = []
    no_launch(monkeypatch, calls)
    bf = torch.bfloat16
    pos = torch.arange(6, dtype=torch.int32)
    qkv = torch.zeros(6, 8, 64, dtype=bf)
    q, k = qkv[:, :4], qkv[:, 4:6]
    ro.rotary(table(), pos, q, k, out=(q, k))
    four = qkv.view(2, 3, 8, 64).transpose(1, 2)
    ro.rotary(table(), pos[:3], four[:, :4], four[:, 4:6], out=(four[:, :4], four[:, 4:6]))
    ro.rotary(table(), pos, q, out=torch.zeros_like(q))
    assert len(calls) == 3
    long = torch.zeros(7, 4, 64, dtype=bf)
    for ins, out in (((long[:6],), long[1:]), ((q, k), (q, q[:, :2])), ((q, q), (q, q)),
                     ((q, k), (qkv[:, 2:6], torch.zeros_like(k))), ((q, k), (torch.zeros_like(q), qkv[:, 3:5])),
                     ((long[:6], long[:6, :2]), (long[:6], torch.zeros(6, 2, 64, dtype=bf)))):
        with pytest.raises(AssertionError, match="overlaps"):
            ro.rotary(table(), pos, *ins, out=out)
    assert len(calls) == 3
    seen = q._version
    ro.rotary(table(), pos, q, out=q)
    assert q._version > seen                            # autograd sees the change


def test_strides_that_reach_the_kernel(monkeypatch):
    calls = []
    no_launch(monkeypatch, calls)
    bf = torch.bfloat16
    q = torch.zeros(5, 4, 64, dtype=bf)
    pos = torch.zeros(5, dtype=torch.int32)
    ro.rotary(table(), pos, q)
    args = calls[-1][4:]                                # behind the table, the name, the function, positions
    assert args[0] == 0 and args[2:6] == (0, 64, 256, 1) and args[11] == 4 and args[12:23] == ro._NONE
    assert args[23:28] == (1, 5, 64, _capi.DTYPE_BF16, False)
    x = torch.zeros(2, 5, 4, 64, dtype=bf).transpose(1, 2)
    ro.rotary(table(), torch.zeros(2, 7, dtype=torch.int32)[:, :5], x, x[:, :2])
    args = calls[-1][4:]
    assert args[0] == 7 and args[2:6] == (1280, 64, 256, 1) and args[7:11] == (1280, 64, 256, 1)
    ro.rotary(table(), pos[:0], q[:0])                  # no token: no launch
    assert len(calls) == 2


def test_backward_turns_what_needs_a_gradient(monkeypatch):
    """One launch over the operand that asks for it, whatever gradients come in; both in one launch where
    both ask."""
    calls = []
    no_launch(monkeypatch, calls)
    bf = torch.bfloat16
    pos = torch.zeros(5, dtype=torch.int32)
    for grads, heads in (((True, False), (4, 0)), ((False, True), (2, 0)), ((True, True), (4, 2))):
        q, k = (torch.zeros(5, h, 64, dtype=bf, requires_grad=g) for h, g in zip((4, 2), grads))
        out = ro.rotary(table(), pos, q, k)
        assert [t.requires_grad for t in out] == [True, True]
        calls.clear()
        leaves = [t for t, g in zip((q, k), grads) if g]
        got = torch.autograd.grad(out, leaves, [torch.zeros_like(t) for t in out])
        assert [g.shape for g in got] == [t.shape for t in leaves]
        args = calls[0][4:]
        assert len(calls) == 1 and (args[11], args[22]) == heads and args[27] is True
    # and to the second order
    q = torch.zeros(5, 4, 64, dtype=bf, requires_grad=True)
    d = [torch.zeros(5, h, 64, dtype=bf, requires_grad=True) for h in (4, 2)]
    gq, = torch.autograd.grad(ro.rotary(table(), pos, q, torch.zeros(5, 2, 64, dtype=bf)), q, d, create_graph=True)
    calls.clear()
    got = torch.autograd.grad(gq, d, torch.zeros_like(q), allow_unused=True)
    assert got[0].shape == d[0].shape and got[1] is None and len(calls) == 1 and calls[0][4:][22] == 0


@pytest.mark.filterwarnings("ignore")
def test_tangents_and_traces_are_refused(monkeypatch):
    no_launch(monkeypatch)
    q, pos = torch.zeros(5, 4, 64, dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int32)
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        d = fw.make_dual(q, torch.ones_like(q))
        for call in (lambda: ro.rotary(table(), pos, d), lambda: ro.rotary(table(), pos, q, d),
                     lambda: ro.rotary(table(), pos, q, out=d)):
            with pytest.raises(AssertionError, match="forward-mode"):
                call()
        ro.rotary(table(), pos, q)

    def traced(x):
        ro.rotary(table(), pos, q + x)
        return x
    with pytest.raises(AssertionError, match="traced"):
        torch.jit.trace(traced, torch.zeros(1, dtype=torch.bfloat16), check_trace=False)


def test_c_refusals():
    lib = _capi.lib()

    def call(turns=16, r=64, attention=1.0, pos=16, q=16, sq=128, qo=16, H=4, k=None, ko=None, Hk=0, B=1, M=5, D=64,
             dtype=0, t=None):
        s = _capi.RotaryStruct(turns=turns, rotary_dim=r, interleaved=0, attention=attention)
        return lib.ugbsa_rotary(ctypes.addressof(s) if t is None else t, pos, 0, q, 0, 64, sq, 1, qo, 0, 64, 256, 1,
                                H, k, 0, 64, 256, 1, ko, 0, 64, 256, 1, Hk, B, M, D, dtype, 0, None)

    def refused(rc, code, word):
        assert rc == code and word in lib.ugbsa_last_error().decode(), (rc, lib.ugbsa_last_error())
    refused(call(t=0), -1, "table")
    refused(call(turns=None), -1, "table")
    refused(call(turns=12), -2, "aligned")
    for r in (0, 63, 66, -2):
        refused(call(r=r), -1, "rotary_dim")
    refused(call(attention=float("nan")), -1, "attention")
    refused(call(D=96), -1, "head_dim")
    refused(call(dtype=5), -3, "dtype")
    refused(call(H=0), -1, "positive")
    refused(call(Hk=-1), -1, "heads")
    refused(call(H=65536), -1, "heads")
    refused(call(M=-1), -1, "B * M")
    refused(call(M=1 << 27), -1, "B * M")
    refused(call(B=1 << 20, M=1 << 20), -1, "B * M")
    refused(call(pos=None), -1, "positions")
    refused(call(pos=18), -1, "positions")
    refused(call(q=None), -1, "q is null")
    refused(call(q=24), -2, "aligned")
    refused(call(sq=100), -2, "strides")
    refused(call(qo=None), -1, "q_out")
    refused(call(Hk=2, ko=16), -1, "k is null")
    refused(call(Hk=2, k=16), -1, "k_out")
    assert call(M=0) == 0
