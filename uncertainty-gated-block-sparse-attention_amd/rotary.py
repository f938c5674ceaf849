"""Rotary positions: queries and keys turned by where their tokens stand, before they are attended
with or cached.

    rot = Rotary.make(128, "cuda", base=1e6, scaling="yarn", factor=4.0, original=32768)
    q, k = rotary(rot, positions, q, k)            # packed tokens [T, H, D], positions [T]
    q, k = rotary(rot, positions, q, k)            # [B, H, M, D], positions [B, M] or [M]
    paged_write(cache, k, v, block_table, seq_lens, cu_new=cu, rotary=rot, positions=positions)

Pair j of a head's first ``rotary_dim`` dims is turned by the angle position * f_j: (j, j + rotary_dim
/ 2), or (2 j, 2 j + 1) where the table is interleaved; the other dims pass unchanged.  Angles are
reduced in 64 bits: cos and sin are off by less than 2^-22 + 2.4 |position| f_j 2^-53, whose second
part is the smaller up to angles of 2^29; the products are fp32, rounded once.  ``rotary`` is
differentiable in q and k.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass, field

import torch
from torch.autograd import forward_ad

import _capi

_tracing_state = torch._C._get_tracing_state


@dataclass(frozen=True, eq=False)
class Rotary:
    """The turns of each pair.  The handle keeps the tensor and its address.

    turns : [rotary_dim / 2] fp64 contiguous on the device, f_j / (2 pi): what pair j turns from one
    position to the next
    interleaved : pairs (2 j, 2 j + 1) instead of (j, j + rotary_dim / 2)
    attention : what the turned values are multiplied by (the factor that goes with some scalings)
    """

    turns: torch.Tensor
    interleaved: bool = False
    attention: float = 1.0
    device: torch.device = field(init=False, default=None)
    _struct: _capi.RotaryStruct = field(init=False, repr=False, compare=False, default=None)
    _call: tuple = field(init=False, repr=False, compare=False, default=None)   # address, device, rotary_dim

    def __post_init__(self):
        t = self.turns
        assert t.dim() == 1 and t.numel() >= 1 and t.dtype == torch.float64 and t.is_contiguous(), \
            "turns [rotary_dim / 2] fp64 contiguous expected"
        assert t.is_cuda and not (t.requires_grad or t.is_neg()), "turns: a HIP tensor without gradients required"
        assert math.isfinite(self.attention), "attention must be finite"
        s = _capi.RotaryStruct(turns=t.data_ptr(), rotary_dim=2 * t.numel(), interleaved=bool(self.interleaved),
                               attention=self.attention)
        object.__setattr__(self, "_struct", s)
        object.__setattr__(self, "device", t.device)
        object.__setattr__(self, "_call", (ctypes.addressof(s), t.get_device(), 2 * t.numel()))

    @classmethod
    def make(cls, rotary_dim, device, base=10000.0, interleaved=False, scaling=None, factor=1.0, original=None,
             fast=32.0, slow=1.0, attention=None):
        """The table of f_j = base^(-2 j / rotary_dim), as it is or scaled for contexts ``factor`` times
        the original:

        "linear" : f_j / factor
        "ntk" : the base grows by factor^(rotary_dim / (rotary_dim - 2)), so the last pair slows by factor
        "yarn" : pairs that turn more than ``fast`` times within ``original`` tokens stay, those that turn
        less than ``slow`` times slow by factor, a ramp between them; attention 0.1 ln(factor) + 1

        ``attention`` overrides that factor.
        """
        f, m = _frequencies(rotary_dim, base, scaling, factor, original, fast, slow)
        turns = torch.tensor([x / (2 * math.pi) for x in f], dtype=torch.float64, device=device)
        return cls(turns, interleaved, m if attention is None else attention)

    @classmethod
    def from_frequencies(cls, frequencies, device=None, interleaved=False, attention=1.0):
        """The table of given f_j [rotary_dim / 2] (radians a position), as model code computes them."""
        f = torch.as_tensor(frequencies, dtype=torch.float64, device=device).detach()
        return cls((f / (2 * math.pi)).contiguous(), interleaved, attention)


def _frequencies(rotary_dim, base, scaling, factor, original, fast, slow):
    """([f_j], attention factor) of ``Rotary.make``."""
    r = rotary_dim
    assert r >= 2 and r % 2 == 0, f"rotary_dim must be even and at least 2, got {r}"
    assert math.isfinite(base) and base > 0, "base must be positive and finite"
    assert scaling in (None, "linear", "ntk", "yarn"), f"unknown scaling {scaling!r}"
    assert math.isfinite(factor) and factor > 0, "factor must be positive and finite"
    assert scaling is not None or factor == 1.0, "factor without a scaling"
    m = 1.0
    if scaling == "ntk":
        assert r > 2, "ntk scaling needs more than one pair"
        base = base * factor ** (r / (r - 2))
    f = [base ** (-2.0 * j / r) for j in range(r // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "yarn":
        assert original is not None and original > 0, "yarn scaling needs the original context length"
        assert base > 1 and fast > slow > 0 and factor >= 1, "yarn scaling needs base > 1, fast > slow > 0, factor >= 1"

        def pair(turns):      # the pair that turns so often within the original context
            return r * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), r - 1)
        ramp = [min(max((j - low) / max(high - low, 0.001), 0.0), 1.0) for j in range(r // 2)]
        f = [x * (1 - w) + x / factor * w for x, w in zip(f, ramp)]
        m = 0.1 * math.log(factor) + 1.0
    return f, m


def _check_unwatched(*tensors):
    """Refuses what would lose or freeze values without an error: a tangent beside a tensor's data, a
    trace that records the calls around a launch."""
    assert _tracing_state() is None, "rotary cannot be traced"
    if forward_ad._current_level >= 0:
        assert all(forward_ad.unpack_dual(t).tangent is None for t in tensors if t is not None), \
            "rotary has no forward-mode derivative"


def _operand(name, t, rot, like):
    """A 16-bit tensor of q's dtype, tokens and head_dim that the kernel reads in place, and its (b, h, m, d)
    strides."""
    assert t.dtype in (torch.bfloat16, torch.float16) and t.dtype is like.dtype, \
        f"{name}: bf16 or fp16 required, q's, got {t.dtype}"
    assert t.get_device() == rot._call[1], f"{name} must be on the table's device"
    st = _strides(t)
    if st[3] == 1 and not (t.data_ptr() & 15 or (st[0] | st[1] | st[2]) & 7 or t.is_neg()):
        return t, st
    if t.is_neg():
        t = t.resolve_neg()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:-1]):
        t = t.clone(memory_format=torch.contiguous_format)
    return t, _strides(t)


def _span(t):
    """[first, last) byte that a tensor's elements reach (its strides are not negative)."""
    last = t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
    return t.data_ptr(), last


def _check_out(outs, ins):
    """Results that the kernel fills in place: what is stored is what the tensor holds, each element has
    a place of its own, and none lies over an input but its own, element on element."""
    for o, x in zip(outs, ins):
        assert o.shape == x.shape and o.dtype is x.dtype and o.get_device() == x.get_device(), \
            "out: tensors like q and k expected"
        assert not o.is_neg() and not (o.requires_grad and torch.is_grad_enabled()), \
            "out: plain tensors without gradients required"
        assert o.stride(-1) == 1 and o.data_ptr() % 16 == 0 and not any(s % 8 for s in o.stride()[:-1]), \
            "out: unit head_dim stride and 16-byte aligned rows required"
        size = 0
        for s, n in sorted((s, n) for s, n in zip(o.stride(), o.shape) if n > 1):
            assert s > size, "out: elements share memory"
            size += (n - 1) * s
    for i, o in enumerate(outs):
        lo, hi = _span(o)
        for j, t in enumerate((*ins, *outs)):
            if j == len(ins) + i or (j == i and t.data_ptr() == o.data_ptr() and t.stride() == o.stride()):
                continue
            a, b = _span(t)
            assert lo >= b or a >= hi or _apart(o, t), "out overlaps another tensor of the call"


def _apart(a, b):
    """Whether two tensors whose ranges overlap are heads side by side in the same tokens (views of one
    projection)."""
    h = a.dim() - (2 if a.dim() == 3 else 3)      # the heads' dimension
    at = [i for i in range(a.dim() - 1) if i != h and a.shape[i] > 1]
    if not at or any(a.stride(i) != b.stride(i) for i in at):
        return False
    token = min(a.stride(i) for i in at)
    if token <= 0 or any(a.stride(i) % token for i in at):
        return False
    wide = [(t.shape[h] - 1) * t.stride(h) + t.shape[-1] for t in (a, b)]
    off = (b.data_ptr() - a.data_ptr()) // a.element_size() % token
    return wide[0] <= off and off + wide[1] <= token


def _strides(t):
    """(b, h, m, d) strides of a tensor of either layout."""
    st = t.stride()
    return st if len(st) == 4 else (0, st[1], st[0], st[2])


def _like(t):
    """A result in t's order of memory where t has one."""
    if 0 in t.stride():
        return torch.empty(t.shape, dtype=t.dtype, device=t.device)
    return torch.empty_like(t)


_NONE = (None, 0, 0, 0, 0, None, 0, 0, 0, 0, 0)


def _launch(rot, what, fn, *args):
    """fn(table, *args, stream) on the table's device."""
    address, index, _ = rot._call
    if torch._C._cuda_getDevice() == index:
        rc = fn(address, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(address, *args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _capi.check(rc, what)


class _Turn(torch.autograd.Function):
    """The gradient of a rotation is the rotation the other way, itself differentiable."""

    @staticmethod
    def forward(ctx, rot, positions, inverse, q, k):
        ctx.rot, ctx.inverse = rot, inverse
        ctx.save_for_backward(positions)
        ctx.set_materialize_grads(False)
        return _turn(rot, positions, q, k, None, inverse)

    @staticmethod
    def backward(ctx, dq, dk=None):
        positions, = ctx.saved_tensors
        # an operand that needs no gradient is not turned back, though its result has one to give
        dq, dk = (d if need else None for d, need in zip((dq, dk), ctx.needs_input_grad[3:]))
        if dq is None and dk is None:
            return None, None, None, None, None
        if dq is None:
            return None, None, None, None, _Turn.apply(ctx.rot, positions, not ctx.inverse, dk, None)
        got = _Turn.apply(ctx.rot, positions, not ctx.inverse, dq, dk)
        return (None, None, None, got, None) if dk is None else (None, None, None, *got)


def _turn(rot, positions, q, k, out, inverse):
    """``rotary`` without gradients."""
    shape = q.shape
    assert len(shape) in (3, 4), "q: [T, H, D] or [B, H, M, D] expected"
    if len(shape) == 3:
        (M, H, D), B = shape, 1
        want = (M,)
    else:
        B, H, M, D = shape
        want = (M,) if positions.dim() == 1 else (B, M)
    assert H >= 1 and B >= 1 and D in (64, 128, 256) and rot._call[2] <= D, \
        f"q: at least one head, head_dim 64, 128 or 256 that holds the table's {rot._call[2]} dims expected"
    assert positions.dtype is torch.int32 and positions.get_device() == rot._call[1], \
        "positions: int32 on the table's device expected"
    assert positions.shape == want, f"positions {list(want)} expected, got {list(positions.shape)}"
    assert M <= 1 or positions.stride(-1) == 1, "positions: a row's entries must be contiguous"
    (qc, q_st), kc, Hk = _operand("q", q, rot, q), None, 0
    if k is not None:
        Hk = k.shape[1] if k.dim() == len(shape) else 0
        assert Hk >= 1 and tuple(k.shape) == ((M, Hk, D) if len(shape) == 3 else (B, Hk, M, D)), \
            f"k {'[T, Hk, D]' if len(shape) == 3 else '[B, Hk, M, D]'} with q's tokens expected, got {list(k.shape)}"
        kc, k_st = _operand("k", k, rot, q)
    if out is None:
        qo, ko = _like(qc), None if k is None else _like(kc)
    else:
        outs = (out,) if torch.is_tensor(out) else tuple(out)
        assert len(outs) == (1 if k is None else 2), "out: a tensor for each of q and k expected"
        _check_out(outs, (q,) if k is None else (q, k))
        for o in outs:
            if not o.is_inference():      # those have no version for autograd to look at
                torch.autograd.graph.increment_version(o)
        qo, ko = (*outs, None)[:2]
    if M:
        kv = _NONE if k is None else (kc.data_ptr(), *k_st, ko.data_ptr(), *_strides(ko), Hk)
        _launch(rot, "rotary", _capi.lib().ugbsa_rotary, positions.data_ptr(),
                positions.stride(0) if len(want) == 2 else 0, qc.data_ptr(), *q_st, qo.data_ptr(),
                *_strides(qo), H, *kv, B, M, D, _capi.dtype_code(q.dtype), inverse)
    return qo if k is None else (qo, ko)


def rotary(rot, positions, q, k=None, out=None, inverse=False):
    """q (and k, in the same launch) turned by their positions.

    q, k : [T, H, D] packed tokens, or [B, H, M, D]; k may have another number of heads
    positions : [T], or [B, M] or [M], int32, any values
    out : the result tensor(s) to fill; an input itself may be given, where it is turned in place
    inverse : by the opposite angles (the result of ``rotary`` back to what it was, but for the table's
    attention factor, which is applied again)

    Returns the turned q, or (q, k) (``out`` if given).  Differentiable in q and k, to any order, unless ``out`` is given.
    Where one of q and k requires a gradient, both results do, and the gradient of the other's is left
    out: ``detach()`` that result before a call that takes none, such as ``paged_write``.
    A backward pass that is captured in a graph needs leaves that no eager graph holds.
    """
    if forward_ad._current_level >= 0 or _tracing_state() is not None:
        _check_unwatched(q, k, *(() if out is None else (out,) if torch.is_tensor(out) else out))
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        assert out is None, "rotary: out has no gradient"
        return _Turn.apply(rot, positions, bool(inverse), q, k)
    return _turn(rot, positions, q, k, out, bool(inverse))
