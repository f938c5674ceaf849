"""Rotary positions against the formula in 64 bits on the same inputs, and their gradients."""

import math
from fractions import Fraction

import pytest
import torch

import rotary as ro

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, FH = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def halves(rot, x):
    r = rot._call[2]
    if rot.interleaved:
        return x[..., 0:r:2], x[..., 1:r:2]
    return x[..., :r // 2], x[..., r // 2:r]


def turned(rot, positions, x, inverse=False):
    """(result, bound of |error| before the last rounding) in fp64; positions broadcast to x[..., 0].

    cos and sin are off by less than 2^-22: 2^-23.3 from the angle's two roundings below pi / 4, 2^-25
    from the series' last sum, as much from what comes before it, 2^-24 from the product with the
    factor; the two products and the sum of a pair add 2^-24 of each term and of the result."""
    x = x.double()
    angle = 2 * math.pi * torch.remainder(positions.double().unsqueeze(-1) * rot.turns, 1.0)
    c, s = rot.attention * torch.cos(angle), rot.attention * torch.sin(angle) * (-1 if inverse else 1)
    a, b = halves(rot, x)
    y, slack = x.clone(), torch.zeros_like(x)
    ya, yb = halves(rot, y)
    ya.copy_(a * c - b * s)
    yb.copy_(b * c + a * s)
    for part in halves(rot, slack):
        part.copy_((a.abs() + b.abs()) * abs(rot.attention) * 2.0 ** -21)
    return y, slack


def check(got, want, slack, extra=1):
    eps = torch.finfo(got.dtype).eps / 2                       # half a step of the result's own rounding
    tiny = torch.finfo(got.dtype).smallest_normal * eps        # and of its subnormals
    err = (got.double() - want).abs()
    assert got.shape == want.shape and (err <= extra * (eps * (want.abs() + slack) + slack + tiny)).all(), err.max()


def table(r, interleaved=False, scaling=None):
    kw = dict(linear=dict(factor=8.0), ntk=dict(factor=8.0), yarn=dict(factor=4.0, original=4096)).get(scaling, {})
    return ro.Rotary.make(r, DEV, interleaved=interleaved, scaling=scaling, **kw)


@pytest.mark.parametrize("T", [1, 2, 65, 333])
@pytest.mark.parametrize("H,Hk,D,r", [(28, 4, 128, 128), (1, 1, 64, 64), (5, 3, 256, 64), (16, 2, 256, 256),
                                      (7, 1, 128, 32), (4, 4, 64, 2), (9, 2, 128, 90), (6, 5, 256, 200)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_packed(hip_lib, T, H, Hk, D, r, interleaved):
    """Heads of one projection, tokens at scattered positions, every layout and share of a head."""
    print(f"[case] packed T={T} H={H}/{Hk} D={D} r={r} {interleaved}", flush=True)
    g = gen(T + H)
    dtype = FH if (T + H) % 2 else BF
    rot = table(r, interleaved, [None, "linear", "yarn"][T % 3])
    qkv = torch.randn(T, H + 2 * Hk, D, generator=g, device=DEV).to(dtype)
    keep = qkv.clone()
    q, k = qkv[:, :H], qkv[:, H:H + Hk]
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=DEV, dtype=torch.int32)
    got = ro.rotary(rot, pos, q, k)
    for x, y in zip((q, k), got):
        check(y, *turned(rot, pos[:, None], x))
        assert torch.equal(y[..., r:], x[..., r:])
    assert torch.equal(qkv, keep)
    assert torch.equal(ro.rotary(rot, pos, q), got[0])
    out = ro.rotary(rot, pos, q, k, out=(q, k))                  # where they are
    assert out[0] is q and torch.equal(q, got[0]) and torch.equal(k, got[1])
    assert torch.equal(qkv[:, H + Hk:], keep[:, H + Hk:])


@pytest.mark.parametrize("B,M", [(1, 1), (3, 1), (2, 65), (3, 1000)])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("dtype,r,interleaved", [(BF, 128, False), (FH, 96, True), (BF, 100, False)])
def test_batched(hip_lib, B, M, shared, dtype, r, interleaved):
    g = gen(B + M)
    rot = table(r, interleaved, "ntk")
    q = torch.randn(B, M, 8, 128, generator=g, device=DEV).to(dtype).transpose(1, 2)
    k = torch.randn(B, 2, M, 128, generator=g, device=DEV).to(dtype)
    pos = torch.randint(0, 40000, (M,) if shared else (B, M + 3), generator=g, device=DEV, dtype=torch.int32)
    pos = pos if shared else pos[:, :M]
    at = pos if shared else pos[:, None]
    for x, y in zip((q, k), ro.rotary(rot, pos, q, k)):
        check(y, *turned(rot, at, x))


def test_many_tokens(hip_lib):
    """The form that holds several heads a thread, an odd number of heads, and its last token."""
    g = gen(3)
    rot, T = table(128), 9001
    x = torch.randn(T, 37, 128, generator=g, device=DEV).to(BF)
    pos = torch.arange(T, device=DEV, dtype=torch.int32) + (1 << 17)
    q, k = ro.rotary(rot, pos, x[:, :32], x[:, 32:])
    for a, y in ((x[:, :32], q), (x[:, 32:], k)):
        check(y, *turned(rot, pos[:, None], a))


@pytest.mark.parametrize("r,interleaved", [(128, True), (100, True), (64, False), (98, False), (36, False)])
def test_calls_of_any_size_agree(hip_lib, r, interleaved):
    """A call that streams past the caches, one with several heads a thread and short ones give the same
    bits; those of the short one are the formula's."""
    g = gen(r)
    T = 23000
    rot = ro.Rotary.make(r, DEV, interleaved=interleaved)
    x = torch.randn(T, 31, 128, generator=g, device=DEV).to(BF)
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=DEV, dtype=torch.int32)
    y = ro.rotary(rot, pos, x)
    assert 2 * x.numel() * 2 > 320 << 20
    for a, b in ((0, 9000), (9000, T), (T - 700, T)):
        assert torch.equal(ro.rotary(rot, pos[a:b], x[a:b]), y[a:b])
    check(y[-700:], *turned(rot, pos[-700:, None], x[-700:]))
    z = x.clone()
    assert torch.equal(ro.rotary(rot, pos, z, out=z), y)


def test_calls_of_several_launches(hip_lib):
    """More rows than a grid has threads for: the bits of calls over some of them, where the launches meet
    and at the ends."""
    def same(rot, pos, x, meet):
        T = x.shape[0]
        parts = [slice(max(a - 300, 0), min(a + 300, T)) for a in (0, *meet, T)]
        for p in parts:
            x[p].normal_(generator=gen(p.start))
        want = [ro.rotary(rot, pos[p], x[p].clone()) for p in parts]
        check(want[-1], *turned(rot, pos[parts[-1], None], x[parts[-1]]))
        assert ro.rotary(rot, pos, x, out=x) is x
        for p, w in zip(parts, want):
            assert torch.equal(x[p], w)
            x[p].zero_()
        step = 1 << 22
        assert not any(x[i:i + step].any() for i in range(0, T, step))
    print("[case] 63 threads a row", flush=True)          # one pair turns, 62 dims pass, a thread each
    T = 70_000_000
    assert T * 63 > 1 << 32
    same(table(2), torch.arange(T, device=DEV, dtype=torch.int32), torch.zeros(T, 1, 64, dtype=BF, device=DEV),
         ((1 << 31) // 63, (1 << 31) // 63 * 2))
    print("[case] 16 threads a row", flush=True)
    T = (1 << 27) + 1000
    same(table(256), torch.arange(T, device=DEV, dtype=torch.int32), torch.zeros(T, 1, 256, dtype=BF, device=DEV),
         (1 << 27,))
    torch.cuda.empty_cache()


def test_far_and_negative_positions(hip_lib):
    """A turn of the first pair is 2 pi positions: 32 bits would not hold the angle."""
    pos = i32([0, 1, -1, -77777, 1 << 20, (1 << 24) + 1, (1 << 31) - 1, -(1 << 31)])
    x = torch.ones(8, 2, 64, device=DEV, dtype=FH)
    x[:, 1] = 0.75
    for rot in (table(64), ro.Rotary.from_frequencies([1.0, 3.5, 0.25, 100.0, 7e-9], DEV, interleaved=True)):
        check(ro.rotary(rot, pos, x), *turned(rot, pos[:, None], x))


def test_far_positions_exactly(hip_lib):
    """Angles from exact rationals: the positions of each frequency whose cosine is nearest to zero, where
    bf16 shows absolute errors of some 2^-24, up to 2^31.  Off by the series' 2^-22 and by 2.4 |pos| f 2^-53
    (the product's rounding 2^-53, the table's 2^-53, its 2 pi's 2^-54.5)."""
    pi = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899863")
    freqs = [1.0, 0.8659643233600653, 3.5, 0.25, 2.0 ** -20]
    rot = ro.Rotary.from_frequencies(freqs, DEV)
    rows = []
    for top in (1 << 12, 1 << 20, 1 << 26, 1 << 30, (1 << 31) - 1):
        for j, f in enumerate(freqs):
            near = [min(max(round((2 * k + 1) * math.pi / (2 * f)), 0), top)
                    for k in range(max(int(top * f / math.pi) - 5000, 0), int(top * f / math.pi))] or [top]
            rest = [abs(Fraction(f) * p / pi % 1 - Fraction(1, 2)) for p in near]
            pos = near[rest.index(min(rest))]
            rows += [(pos, j), (-pos, j)]
    pos = i32([p for p, _ in rows])
    x = torch.zeros(len(rows), 1, 64, dtype=BF, device=DEV)
    x[..., :len(freqs)] = 1
    y = ro.rotary(rot, pos, x)[:, 0].double().cpu()
    for i, (p, j) in enumerate(rows):
        angle = float(Fraction(freqs[j]) * p % (2 * pi))
        for got, want in ((y[i, j].item(), math.cos(angle)), (y[i, j + len(freqs)].item(), math.sin(angle))):
            slack = 2.0 ** -22 + 2.4 * abs(p) * freqs[j] * 2.0 ** -53
            # bf16's half step: 2^-8 of values in [.5, 1) apart are 2^-9 off at most, which is 2^-8 of .5
            assert abs(got - want) <= 2.0 ** -8 * (abs(want) + slack) + slack, (p, freqs[j], got, want)


def test_unusual_operands(hip_lib):
    """Negated and misaligned views, odd strides, a stride of 0, an inner stride."""
    g = gen(4)
    rot, pos = table(64), i32([5, 900, 31])
    flat = torch.randn(8192, generator=g, device=DEV).to(BF)
    views = [torch._neg_view(flat[:768].view(3, 4, 64)), flat[4:772].view(3, 4, 64), flat[:3 * 260].view(3, 260)[:, :256].view(3, 4, 64),
             flat[:192].view(3, 1, 64).expand(3, 4, 64), flat[:1536].view(3, 4, 128)[..., ::2], flat[:768].view(3, 64, 4).transpose(1, 2)]
    for v in views:
        check(ro.rotary(rot, pos, v), *turned(rot, pos[:, None], v))
    assert ro.rotary(rot, pos[:0], flat[:0].view(0, 4, 64)).shape == (0, 4, 64)


def test_values_without_a_number(hip_lib):
    """NaN and infinities stay in their pair; dims that pass keep their bits."""
    for interleaved in (False, True):
        rot = table(32, interleaved)
        x = torch.ones(2, 2, 64, device=DEV, dtype=BF)
        x[0, 0, 3], x[0, 1, 20], x[1, 0, 40], x[1, 1, 63] = NAN, INF, NAN, -INF
        y = ro.rotary(rot, i32([0, 9]), x)
        assert torch.equal(y[..., 32:].contiguous().view(torch.int16), x[..., 32:].contiguous().view(torch.int16))
        bad = ~y[..., :32].isfinite()
        want = torch.zeros_like(bad)
        for h, j in ((0, 3), (1, 20)):
            other = (j ^ 1) if interleaved else (j + 16) % 32
            want[0, h, j] = want[0, h, other] = True
        assert torch.equal(bad, want)


def test_inverse_undoes(hip_lib):
    g = gen(5)
    rot = table(128, True)
    x = torch.randn(50, 4, 128, generator=g, device=DEV).to(FH)
    pos = torch.randint(0, 99999, (50,), generator=g, device=DEV, dtype=torch.int32)
    y = ro.rotary(rot, pos, x)
    check(ro.rotary(rot, pos, y, inverse=True), *turned(rot, pos[:, None], y, inverse=True))


# ---- gradients ----------------------------------------------------------------------------------

@pytest.mark.parametrize("interleaved,r", [(False, 128), (True, 64), (False, 36)])
def test_gradient_is_the_formulas(hip_lib, interleaved, r):
    """The transpose of the rotation, for packed, batched and broadcast operands and gradients."""
    g = gen(r)
    rot = table(r, interleaved, "yarn")
    pos = torch.randint(0, 99999, (33,), generator=g, device=DEV, dtype=torch.int32)
    q = torch.randn(2, 33, 6, 128, generator=g, device=DEV).to(BF).transpose(1, 2).requires_grad_()
    k = torch.randn(2, 2, 33, 128, generator=g, device=DEV).to(BF).requires_grad_()
    dq = torch.randn(2, 6, 33, 128, generator=g, device=DEV).to(BF)
    dk = torch.randn(2, 1, 1, 128, generator=g, device=DEV).to(BF).expand(2, 2, 33, 128)
    yq, yk = ro.rotary(rot, pos, q, k)
    check(yq.detach(), *turned(rot, pos, q.detach()))
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk), retain_graph=True)
    check(gq, *turned(rot, pos, dq, inverse=True))
    check(gk, *turned(rot, pos, dk, inverse=True))
    # one of the two alone, and a key without a gradient
    assert torch.equal(torch.autograd.grad(yq, q, dq, retain_graph=True)[0], gq)
    assert torch.equal(torch.autograd.grad(yk, k, dk)[0], gk)
    yq, yk = ro.rotary(rot, pos, q, k.detach())
    assert torch.equal(torch.autograd.grad((yq, yk), q, (dq, dk))[0], gq)
    assert torch.equal(torch.autograd.grad(ro.rotary(rot, pos, k), k, dk)[0], gk)


def test_gradient_by_differences(hip_lib):
    """A linear map: its gradient along v is the difference of two results, exactly but for rounding."""
    g = gen(6)
    rot, pos = table(64), i32([3, 700, 12345])
    x = torch.randint(-8, 9, (3, 2, 64), generator=g, device=DEV).to(FH).requires_grad_()
    v = torch.randint(-8, 9, (3, 2, 64), generator=g, device=DEV).to(FH)
    w = torch.randint(-8, 9, (3, 2, 64), generator=g, device=DEV).to(FH)
    gx, = torch.autograd.grad(ro.rotary(rot, pos, x), x, w)
    with torch.no_grad():
        diff = ro.rotary(rot, pos, x + v).double() - ro.rotary(rot, pos, x).double()
    # results up to 16 * 2^.5 < 32, off by half a step (2^-11 of 32) each, times |w| <= 8, over 64 dims
    # of a head; the gradient's entries up to 8 * 2^.5 < 16, off by 2^-11 of 16, times |v| <= 8
    bound = 64 * (2 * 32 * 2.0 ** -11 * 8 + 16 * 2.0 ** -11 * 8)
    lhs, rhs = (w.double() * diff).sum(-1), (gx.double() * v.double()).sum(-1)
    assert (lhs - rhs).abs().max() <= bound and (lhs.abs().max() > 8 * bound or lhs.abs().max() > 200)


def test_second_derivative(hip_lib):
    """The gradient is differentiable in the gradient it came from."""
    g = gen(7)
    rot, pos = table(128), i32([17, 4000])
    q = torch.randn(2, 4, 128, generator=g, device=DEV).to(BF).requires_grad_()
    d = torch.randn(2, 4, 128, generator=g, device=DEV).to(BF).requires_grad_()
    gq, = torch.autograd.grad(ro.rotary(rot, pos, q), q, d, create_graph=True)
    e = torch.randn(2, 4, 128, generator=g, device=DEV).to(BF)
    gd, = torch.autograd.grad(gq, d, e)
    check(gd, *turned(rot, pos[:, None], e))


def test_gradient_reaches_shared_tensors(hip_lib):
    """q and k of one projection, and a tensor turned by two tables, get the sum of their gradients."""
    g = gen(8)
    a, b, pos = table(64), table(64, True), i32([4, 9, 100])
    x = torch.randn(3, 6, 64, generator=g, device=DEV).to(BF).requires_grad_()
    dq, dk = (torch.randn(3, h, 64, generator=g, device=DEV).to(BF) for h in (4, 2))
    gx, = torch.autograd.grad(ro.rotary(a, pos, x[:, :4], x[:, 4:]), x, (dq, dk))
    check(gx, *(torch.cat(p, 1) for p in zip(turned(a, pos[:, None], dq, True), turned(a, pos[:, None], dk, True))))
    y = ro.rotary(a, pos, x), ro.rotary(b, pos, x)
    d = torch.randn(3, 6, 64, generator=g, device=DEV).to(BF)
    gx, = torch.autograd.grad(y, x, (d, d))
    one, two = turned(a, pos[:, None], d, True), turned(b, pos[:, None], d, True)
    # each rounded to bf16, then their sum
    err = (gx.double() - one[0] - two[0]).abs()
    assert (err <= 2.0 ** -8 * 1.01 * (one[0].abs() + two[0].abs() + (one[0] + two[0]).abs()) + 1e-5).all()


# ---- streams and graphs -------------------------------------------------------------------------

def test_on_another_stream(hip_lib):
    g = gen(9)
    rot = table(128)
    x = torch.randn(300, 8, 128, generator=g, device=DEV).to(BF)
    pos = torch.arange(300, device=DEV, dtype=torch.int32)
    want = ro.rotary(rot, pos, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ro.rotary(rot, pos, x)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("grad", [False, True])
def test_replayed(hip_lib, grad):
    """A captured turn, and its backward pass, follow what their tensors hold at each replay."""
    g = gen(10)
    rot = table(64, scaling="yarn")
    x = torch.randn(40, 6, 64, generator=g, device=DEV).to(BF)
    d = torch.randn(40, 6, 64, generator=g, device=DEV).to(BF)
    pos = torch.arange(40, device=DEV, dtype=torch.int32)

    def step():
        leaf = x.detach().requires_grad_(grad)
        y = ro.rotary(rot, pos, leaf)
        return (y, *torch.autograd.grad(y, leaf, d)) if grad else (y,)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        pos += 1000
        x.mul_(-0.5)
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.detach(), b)
