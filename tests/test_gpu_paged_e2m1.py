"""The paged cache in four bits: writing, reading back and decode attention against 64-bit references
on the same inputs; keys turned on the way into any cache."""

import math

import pytest
import torch

import paged_cache as pc
import rotary as ro
from test_gpu_paged_cache import bits, bound, check_close, gen, i32, tables

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, FH = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---- e2m1 by its definition ---------------------------------------------------------------------

def e2m1_ref(x, dtype):
    """(values of the codes [..., D], scale bytes [..., D / 32]) of x [..., D] fp64: the nearest of the
    eight magnitudes, of two as near the one of the even code; the scale the smallest power of two with
    max |x| <= 6 scale over 32 dims; all NaN, byte 255, where one of them is."""
    top = 1.5 * 2.0 ** (15 if dtype == FH else 127)
    x = x.unflatten(-1, (-1, 32)).clamp(-top, top)
    mx = torch.nan_to_num(x, nan=0.0).abs().amax(-1)
    e = [0 if m == 0 else max(math.frexp(m)[1] - 3 + (math.frexp(m)[0] > 0.75), -127) for m in mx.flatten().tolist()]
    e = torch.tensor(e, dtype=torch.float64, device=x.device).view(mx.shape)
    y = (x * torch.exp2(-e).unsqueeze(-1)).abs()
    best = torch.zeros_like(y)
    for i, v in enumerate(GRID):
        d, old = (y - v).abs(), (y - best).abs()
        best = torch.where((d < old) | ((d == old) & (i % 2 == 0)), v, best)
    nan = x.isnan().any(-1)
    val = (best * x.sign()).masked_fill(nan.unsqueeze(-1), NAN)
    byte = (e + 127).masked_fill(nan, 255).to(torch.uint8)
    return val.flatten(-2), byte


def cache_values(cache, name):
    """The pool of an e2m1 cache as fp64 values [P, Hk, 64, D]."""
    codes = getattr(cache, name + "_pages")
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    x = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device=DEV)[both]
    byte = getattr(cache, name + "_scale").transpose(2, 3)
    scale = torch.exp2(byte.double() - 127).masked_fill(byte == 255, NAN)
    return x * scale.repeat_interleave(32, -1)


def filled(g, P, Hk, D, dtype, interleaved=False):
    """A cache of random codes, keys and values of about 1."""
    if interleaved:       # K and V of a page side by side in one pool
        pool = torch.empty(P, 2, Hk, 64, D // 2, dtype=torch.uint8, device=DEV)
        sc = [torch.empty(P, Hk, D // 32, 64, dtype=torch.uint8, device=DEV) for _ in range(2)]
        cache = pc.PagedCache(pool[:, 0], pool[:, 1], *sc, torch.empty(P, Hk, 2, D, dtype=dtype, device=DEV), dtype)
    else:
        cache = pc.PagedCache.empty(P, Hk, D, dtype, DEV, e2m1=True)
    for t in (cache.k_pages, cache.v_pages):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=DEV))
    for t in (cache.k_scale, cache.v_scale):
        t.copy_(torch.randint(124, 127, t.shape, generator=g, device=DEV))
    mid = torch.randn(P, Hk, D, generator=g, device=DEV)
    cache.planes.copy_(torch.stack([mid + 1.5, mid - 1.5], 2))
    return cache


SHAPES = [(8, 8, 64, BF), (8, 2, 64, FH), (28, 4, 128, BF), (34, 2, 128, FH), (16, 2, 256, BF), (9, 1, 256, FH),
          (40, 2, 128, BF), (7, 1, 64, FH)]


# ---- write and read -----------------------------------------------------------------------------

def stored(cache, x, name, page, slot):
    """(values of codes, bytes) of one head's token rows [T, Hk] as they lie in the cache."""
    val = cache_values(cache, name)[page, :, slot]
    return val, getattr(cache, name + "_scale")[page, :, :, slot]


@pytest.mark.parametrize("lens,new", [([0], [1]), ([63], [1]), ([5, 0, 130], [0, 70, 1]), ([0, 1, 63, 64], [64, 63, 2, 200])])
@pytest.mark.parametrize("Hk,D,dtype", [(4, 128, BF), (2, 64, FH), (1, 256, BF), (3, 256, FH), (2, 64, BF)])
def test_write_and_read(hip_lib, lens, new, Hk, D, dtype):
    print(f"[case] e2m1 write {lens} {new} Hk={Hk} D={D} {dtype}", flush=True)
    g = gen(D + Hk + len(lens))
    table, P = tables([a + b for a, b in zip(lens, new)], g)
    cache = filled(g, P, Hk, D, dtype, interleaved=D == 128)
    T = sum(new)
    kv = torch.randn(T + 3, 2, Hk, D, generator=g, device=DEV) * torch.exp(
        2 * torch.randn(T + 3, 2, Hk, D // 32, 1, generator=g, device=DEV)).expand(-1, -1, -1, -1, 32).flatten(-2)
    kv = kv.to(dtype)
    before = {n: getattr(cache, n).clone() for n in ("k_pages", "v_pages", "k_scale", "v_scale", "planes")}
    cu = i32([sum(new[:i]) for i in range(len(new) + 1)])
    pc.paged_write(cache, kv[:, 0], kv[:, 1], table, i32(lens), cu_new=cu)
    rows, touched = table.tolist(), torch.zeros(P, 64, dtype=torch.bool, device=DEV)
    planes, at = before["planes"].double(), 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for i in range(m):
            page, slot = rows[b][(n + i) // 64], (n + i) % 64
            touched[page, slot] = True
            if slot == 0:
                planes[page, :, 0], planes[page, :, 1] = -INF, INF
            key = kv[at + i, 0].double()
            planes[page, :, 0] = torch.maximum(planes[page, :, 0], key)
            planes[page, :, 1] = torch.minimum(planes[page, :, 1], key)
        pos = torch.arange(n, n + m, device=DEV)
        page, slot = table[b].long()[pos // 64], pos % 64
        for j, name in enumerate("kv"):
            val, byte = e2m1_ref(kv[at:at + m, j].double(), dtype)
            got, gotb = stored(cache, kv, name, page, slot)
            assert torch.equal(gotb, byte)
            assert torch.equal(got, val * torch.exp2(byte.double() - 127).repeat_interleave(32, -1))
        at += m
    assert torch.equal(cache.planes.double(), planes)
    for name in ("k", "v"):                                      # the other slots keep their bits
        keep = ~touched.view(P, 1, 64, 1).expand_as(cache.k_pages)
        assert torch.equal(getattr(cache, name + "_pages")[keep], before[name + "_pages"][keep])
        keep = ~touched.view(P, 1, 1, 64).expand_as(cache.k_scale)
        assert torch.equal(getattr(cache, name + "_scale")[keep], before[name + "_scale"][keep])
    after = [a + b for a, b in zip(lens, new)]
    for n in (max(after), max(after) + 70, max(1, min(after))):
        for name, t in zip("kv", pc.paged_read(cache, table, i32(after), n)):
            want = torch.zeros(len(lens), Hk, n, D, dtype=torch.float64, device=DEV)
            vals = cache_values(cache, name)
            for b, m in enumerate(after):
                pos = torch.arange(min(m, n), device=DEV)
                want[b, :, :min(m, n)] = vals[table[b].long()[pos // 64], :, pos % 64].transpose(0, 1)
            assert torch.equal(t.double(), want)                 # exact in the model's dtype


def test_special_values(hip_lib):
    """Zeros, halves, subnormals, the largest values, infinities and NaN, each in a group of its own."""
    for dtype, big in ((FH, 65504.0), (BF, 3.3895e38)):
        rows = [[0.0] * 32, [-0.0] * 32, [big] + [1.0] * 31, [-big] + [big / 3] * 31, [INF, -INF] + [2.0] * 30,
                [NAN, 1.0, -448.0] + [0.5] * 29, [INF, NAN] + [1.0] * 30, [NAN] * 32, [6e-8] * 32,
                [6e-8, 1.2e-7] + [3e-7] * 30, [6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25] * 4,
                [-6.0, -5.0, -3.5, -2.5, -1.75, -1.25, -0.75, -0.25] * 4, [6.0, 0.2, 0.26, 2.4, 2.6] + [5.1] * 27,
                [12.0, 11.9, 7.0, 0.49] + [0.51] * 28, [6.03125, 3.0] + [1.0] * 30, [49152.0] + [3.0] * 31,
                [1.0] + [2.0 ** -14] * 31, [1e-3] * 32]
        if dtype == BF:
            rows += [[1e-40] * 32, [9.2e-41, 1.8e-40] + [0.0] * 30, [1.2e-38] + [1e-39] * 31, [2.4e38] + [3e38] * 31]
        x = torch.tensor(rows, device=DEV).to(dtype)
        x = torch.cat([x, x.flip(0)], 1).view(len(rows), 1, 64)
        cache = pc.PagedCache.empty(1, 1, 64, dtype, DEV, e2m1=True)
        pc.paged_write(cache, x, x, i32([[0]]), i32([0]), cu_new=i32([0, len(rows)]))
        val, byte = e2m1_ref(x.double(), dtype)
        want = (val * torch.exp2(byte.double() - 127).repeat_interleave(32, -1))[:, 0]
        k, v = pc.paged_read(cache, i32([[0]]), i32([len(rows)]), len(rows))
        for name, t in (("k", k), ("v", v)):
            assert torch.equal(getattr(cache, name + "_scale")[0, 0, :, :len(rows)].T, byte[:, 0])
            assert torch.equal(cache_values(cache, name)[0, 0, :len(rows)].nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))
            assert torch.equal(t[0, 0].double().nan_to_num(nan=-7.0), want.nan_to_num(nan=-7.0))
        assert torch.isposinf(cache.planes[0, 0, 0, 0]) and not cache.planes.isnan().any()


@pytest.mark.parametrize("kind", ["model", "e4m3", "e2m1"])
@pytest.mark.parametrize("D,r,interleaved", [(128, 128, False), (64, 64, True), (256, 64, False), (128, 90, False),
                                             (256, 130, True), (64, 2, False)])
@pytest.mark.parametrize("own_positions", [False, True])
def test_keys_turned_on_the_way(hip_lib, kind, D, r, interleaved, own_positions):
    """The bits that turning them first and writing them then gives."""
    g = gen(D + r)
    dtype = FH if r % 4 else BF
    lens, new = [0, 63, 200], [130, 2, 1]
    table, P = tables([a + b for a, b in zip(lens, new)], g)
    T = sum(new)
    qkv = torch.randn(T + 2, 6, D, generator=g, device=DEV).to(dtype)
    k, v = qkv[:, 2:4], qkv[:, 4:]
    rot = ro.Rotary.make(r, DEV, interleaved=interleaved, scaling="linear", factor=2.0)
    place = [n + i for n, m in zip(lens, new) for i in range(m)] + [0, 0]
    pos = torch.randint(0, 1 << 20, (T + 2,), generator=g, device=DEV, dtype=torch.int32) if own_positions else i32(place)
    cu = i32([sum(new[:i]) for i in range(4)])
    caches = []
    for _ in range(2):
        cache = pc.PagedCache.empty(P, 2, D, dtype, DEV, e4m3=kind == "e4m3", e2m1=kind == "e2m1")
        for n in ("k_pages", "v_pages", "k_scale", "v_scale", "planes"):
            if getattr(cache, n) is not None:
                getattr(cache, n).view(torch.uint8).fill_(3)
        caches.append(cache)
    keep = qkv.clone()
    pc.paged_write(caches[0], k, v, table, i32(lens), cu_new=cu, rotary=rot, positions=pos if own_positions else None)
    pc.paged_write(caches[1], ro.rotary(rot, pos, k), v, table, i32(lens), cu_new=cu)
    assert torch.equal(qkv, keep)
    for n in ("k_pages", "v_pages", "k_scale", "v_scale", "planes"):
        if getattr(caches[0], n) is not None:
            assert torch.equal(bits(getattr(caches[0], n)), bits(getattr(caches[1], n))), n
    # one token each
    pc.paged_write(caches[0], k[:3], v[:3], table, i32([10, 20, 30]), rotary=rot)
    pc.paged_write(caches[1], ro.rotary(rot, i32([10, 20, 30]), k[:3]), v[:3], table, i32([10, 20, 30]))
    assert torch.equal(bits(caches[0].k_pages), bits(caches[1].k_pages))


# ---- decode -------------------------------------------------------------------------------------

def decode_ref(q, cache, table, lens, scale, kv_idx=None, counts=None):
    """(out, sum of p |v|, the largest sum of |q_d k_d|, sum of |v|) [B, 1, H, D] fp64 by the definition."""
    B, H, _, D = q.shape
    Hk, NB = cache.k_scale.shape[1], table.shape[1]
    P = cache.k_pages.shape[0]
    # what paged_read gives: values past the range of the model's dtype, which paged_write does not
    # store, are rounded to it
    kc, vc = (cache_values(cache, n).to(q.dtype).double() for n in "kv")
    out = torch.zeros(2, B, 1, H, D, dtype=torch.float64, device=DEV)
    size, flat = torch.zeros(B, 1, H, 1, dtype=torch.float64, device=DEV), torch.zeros_like(out[0])
    for b in range(B):
        n = min(max(lens[b], 0), 64 * NB)
        for h in range(Hk):
            blocks = range(NB) if kv_idx is None else kv_idx[b, h, :kv_idx.shape[2] if counts is None else
                                                            max(int(counts[b, h]), 0)].tolist()
            blocks = [j for j in blocks if 0 <= j < NB and 64 * j < n and 0 <= int(table[b, j]) < P]
            if not blocks:
                continue
            at = torch.tensor(blocks, device=DEV)
            pages = table[b][at].long()
            live = ((at.view(-1, 1) * 64 + torch.arange(64, device=DEV)) < n).flatten()
            k, v = kc[pages, h].flatten(0, 1)[live], vc[pages, h].flatten(0, 1)[live]
            hs = slice(h * (H // Hk), (h + 1) * (H // Hk))
            p = torch.softmax((q[b, hs, 0].double() @ k.T) * scale, -1)
            out[0, b, 0, hs], out[1, b, 0, hs] = p @ v, p @ v.abs()
            # |scale| sum_d |q_d k_d| of the key where it is largest
            size[b, 0, hs, 0] = ((q[b, hs, 0].double().abs() @ k.abs().T) * abs(scale)).amax(-1)
            flat[b, 0, hs] = v.abs().sum(0)
    return out[0], out[1], size, flat


def check_decode(q, cache, table, lens, scale, large=False, **lists):
    """large: for scores of hundreds.  fp32 holds a score to 2^-20 of S = |scale| sum |q_d k_d|: eight
    products of 32 dims added one behind the other (2^-21 S), two roundings of the factor and its
    product, one of the difference to the maximum (2^-24 S each); the weight and the normaliser are off
    by as much of themselves.  Most weights are then next to nothing: fp16 holds one below its normal
    range to 2^-25 of the largest (the normaliser is no smaller), bf16 all to half a step."""
    out = pc.paged_decode(q, cache, table, i32(lens), scale, **lists)
    assert out.shape == (q.shape[0], 1, q.shape[1], q.shape[3]) and out.is_contiguous()
    ref, mass, size, flat = decode_ref(q, cache, table, lens, scale, **lists)
    if large:
        most = bound(ref, mass, q.dtype) + mass * 2 * 2.0 ** -20 * size + (2.0 ** -25 * flat if q.dtype == FH else 0)
        off = (out.double() - ref).abs() / most
        assert off.max() <= 1.0, off.max()
    else:
        check_close(out, ref, mass, q.dtype)
    return out


def poison(cache, table, lens):
    """NaN in every slot that holds no token of a sequence."""
    P = cache.k_pages.shape[0]
    dead = torch.ones(P, 64, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        for j in range((n + 63) // 64):
            dead[table[b, j], : n - 64 * j] = False
    for t in (cache.k_scale, cache.v_scale):
        t.masked_fill_(dead.view(P, 1, 1, 64), 255)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("D,r", [(64, 64), (64, 16), (64, 48), (128, 128), (128, 48), (256, 256), (256, 16), (256, 176)])
def test_keys_whose_lanes_share_their_turns(hip_lib, D, r, dtype):
    """Halves of whole vectors, from the ends of a page and one token a sequence: the bits of ``rotary``."""
    g = gen(D + r)
    rot = ro.Rotary.make(r, DEV, base=500.0, attention=1.3)
    for lens, new in (([0, 63, 200, 7], [64, 2, 77, 1]), ([5, 63, 0, 128], None)):
        T = 4 if new is None else sum(new)
        table, P = tables([a + b for a, b in zip(lens, new or [1] * 4)], g)
        cu = None if new is None else i32([sum(new[:i]) for i in range(5)])
        k, v = (torch.randn(T, 3, D, generator=g, device=DEV).to(dtype) for _ in range(2))
        pos = torch.randint(-(1 << 31), (1 << 31) - 1, (T,), generator=g, device=DEV).to(torch.int32)
        kw = dict(dtype=dtype, device=DEV)
        caches = [pc.PagedCache.empty(P, 3, D, **kw) for _ in range(2)]
        for cache in caches:
            cache.k_pages.zero_(), cache.v_pages.zero_(), cache.planes.zero_()
        pc.paged_write(caches[0], k, v, table, i32(lens), cu_new=cu, rotary=rot, positions=pos)
        pc.paged_write(caches[1], ro.rotary(rot, pos, k), v, table, i32(lens), cu_new=cu)
        for n in ("k_pages", "v_pages", "planes"):
            assert torch.equal(bits(getattr(caches[0], n)), bits(getattr(caches[1], n)))


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("r,interleaved", [(128, False), (48, False), (128, True), (90, False)])
def test_keys_turned_without_a_number(hip_lib, r, interleaved, dtype):
    """Infinities, NaN and zeros of either sign among the keys: what ``rotary`` makes of them, NaN where it has one."""
    g = gen(r)
    rot = ro.Rotary.make(r, DEV, interleaved=interleaved)
    special = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1.0, -2.0, 0.5], device=DEV)
    k = special[torch.randint(0, 8, (100, 2, 128), generator=g, device=DEV)].to(dtype)
    pos = torch.randint(0, 1000, (100,), generator=g, device=DEV).to(torch.int32)
    pos[::3] = 0
    table = i32([[0, 1]])
    caches = [pc.PagedCache.empty(2, 2, 128, dtype, DEV) for _ in range(2)]
    for cache in caches:
        cache.k_pages.zero_(), cache.v_pages.zero_(), cache.planes.zero_()
    cu = i32([0, 100])
    pc.paged_write(caches[0], k, k, table, i32([0]), cu_new=cu, rotary=rot, positions=pos)
    pc.paged_write(caches[1], ro.rotary(rot, pos, k), k, table, i32([0]), cu_new=cu)
    for n in ("k_pages", "v_pages", "planes"):
        x, y = (getattr(c, n) for c in caches)
        assert torch.equal(x.isnan(), y.isnan())
        if n != "planes":
            assert torch.equal(bits(x.masked_fill(x.isnan(), 7.0)), bits(y.masked_fill(y.isnan(), 7.0)))
        else:
            assert torch.equal(x.nan_to_num(nan=7.0), y.nan_to_num(nan=7.0))


@pytest.mark.parametrize("lens", [[1], [0, 31, 32, 33, 63, 64, 65], [511, 0, 1000, 2], [4097], [300] * 40,
                                  [130, 0, 256, 1] * 33])
@pytest.mark.parametrize("H,Hk,D,dtype", SHAPES)
def test_decode(hip_lib, lens, H, Hk, D, dtype):
    print(f"[case] e2m1 decode {lens[:7]} H={H}/{Hk} D={D} {dtype}", flush=True)
    g = gen(D + H + len(lens))
    table, P = tables(lens, g)
    cache = filled(g, P, Hk, D, dtype, interleaved=H == 28)
    poison(cache, table, lens)
    q = torch.randn(len(lens), 1, H, D, generator=g, device=DEV).to(dtype).transpose(1, 2)
    check_decode(q, cache, table, lens, D ** -0.5)


@pytest.mark.parametrize("H,Hk,D,dtype", SHAPES)
def test_decode_wide_tables(hip_lib, H, Hk, D, dtype):
    """Short sequences in tables that ask for the line, and for streaming loads."""
    g = gen(D + H)
    lens = [70, 0, 5, 3000]
    for width in (100, 60000):
        table, P = tables(lens, g, width=width)
        cache = filled(g, P, Hk, D, dtype)
        poison(cache, table, lens)
        q = torch.randn(4, H, 1, D, generator=g, device=DEV).to(dtype)
        check_decode(q, cache, table, lens, D ** -0.5)


@pytest.mark.parametrize("H,Hk,D,dtype", SHAPES)
def test_decode_listed(hip_lib, H, Hk, D, dtype):
    g = gen(D + H + 1)
    lens = [64 * 40 - 5, 3, 64 * 9]
    table, P = tables(lens, g)
    cache = filled(g, P, Hk, D, dtype)
    q = torch.randn(3, H, 1, D, generator=g, device=DEV).to(dtype)
    NB = table.shape[1]
    for slots in (1, 7, 45):
        order = torch.rand(3, Hk, NB, generator=g, device=DEV).argsort(-1)[..., :slots]
        idx = torch.full((3, Hk, slots), NB, dtype=torch.int32, device=DEV)
        idx[..., :order.shape[-1]] = order.to(torch.int32)
        counts = torch.randint(-1, slots + 3, (3, Hk), generator=g, device=DEV, dtype=torch.int32)
        check_decode(q, cache, table, lens, D ** -0.5, kv_idx=idx)
        check_decode(q, cache, table, lens, D ** -0.5, kv_idx=idx, counts=counts.clamp(max=slots))
        pc.paged_decode(q, cache, table, i32(lens), D ** -0.5, kv_idx=idx, counts=counts)


def test_decode_absent_pages_and_lengths(hip_lib):
    g = gen(11)
    cache = filled(g, 6, 2, 128, BF)
    q = torch.randn(4, 8, 1, 128, generator=g, device=DEV).to(BF)
    check_decode(q, cache, i32([[0, -1, 7, 2], [5, 1, 6, -9], [-1, -1, -1, -1], [3, 4, 0, 1]]), [256, 90, 200, 1 << 30], 0.09)
    assert (pc.paged_decode(q, cache, i32([[0]] * 4), i32([-3, 0, 0, -1]), 0.1) == 0).all()


def test_decode_sharp_and_large_scores(hip_lib):
    """One key that takes all the weight, queries far apart in magnitude within a head, and tiny scales."""
    g = gen(12)
    for D, dtype in ((64, BF), (128, BF), (256, FH), (64, FH), (128, FH)):
        lens = [500, 64]
        table, P = tables(lens, g)
        cache = filled(g, P, 2, D, dtype)
        q = torch.randn(2, 10, 1, D, generator=g, device=DEV)
        check_decode((q * 30).to(dtype), cache, table, lens, 1.0, large=True)
        mixed = q * torch.exp2(torch.randint(-12, 4, q.shape, generator=g, device=DEV).float())
        check_decode(mixed.to(dtype), cache, table, lens, 0.5, large=True)
        one = torch.zeros_like(q)
        one[..., 5], one[..., D - 1] = 3.0, 2.0 ** -9
        check_decode(one.to(dtype), cache, table, lens, -1.0)
        cache.k_scale.fill_(100), cache.v_scale.fill_(110)
        check_decode((q * 1000).to(dtype), cache, table, lens, 1000.0)


def test_decode_special_queries(hip_lib):
    """Infinities and NaN stay in their head's row; a zero query weighs all keys alike."""
    g = gen(13)
    table, P = tables([200], g)
    for D, dtype in ((128, BF), (64, FH), (256, BF)):
        cache = filled(g, P, 1, D, dtype)
        q = torch.randn(1, 5, 1, D, generator=g, device=DEV).to(dtype)
        q[0, 1, 0, 3], q[0, 3, 0, 7], q[0, 4] = NAN, INF, 0.0
        out = pc.paged_decode(q, cache, table, i32([200]), 0.1)
        assert out[0, 0, 1].isnan().all() and out[0, 0, 3].isnan().all()
        ref, mass, *_ = decode_ref(q, cache, table, [200], 0.1)
        for h in (0, 2, 4):
            check_close(out[0, 0, h], ref[0, 0, h], mass[0, 0, h], dtype)


def test_decode_of_nan_groups(hip_lib):
    """A key group that is NaN makes every row of its KV head NaN, a value group its 32 dims."""
    g = gen(14)
    table, P = tables([200], g)
    cache = filled(g, P, 2, 128, BF)
    q = torch.randn(1, 4, 1, 128, generator=g, device=DEV).to(BF)
    cache.v_scale[table[0, 1].long(), 0, 2, 9] = 255
    out = pc.paged_decode(q, cache, table, i32([200]), 0.1)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[0, 0, :2, 64:96] = True
    assert torch.equal(out.isnan(), bad)
    cache.k_scale[table[0, 2].long(), 1, 0, 3] = 255
    assert pc.paged_decode(q, cache, table, i32([200]), 0.1)[0, 0, 2:].isnan().all()


def test_pages_past_32_bit_offsets(hip_lib):
    """Pages whose byte offsets need more than 32 bits."""
    g = gen(15)
    Hk, D = 8, 256
    P = (1 << 32) // (Hk * 64 * D // 2) + 40
    k, v = (torch.zeros(P, Hk, 64, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2))
    sc = [torch.full((P, Hk, D // 32, 64), 126, dtype=torch.uint8, device=DEV) for _ in range(2)]
    far = list(range(P - 20, P))
    small = filled(g, 20, Hk, D, BF)
    for t, s in zip((k, v, *sc), (small.k_pages, small.v_pages, small.k_scale, small.v_scale)):
        t[P - 20:] = s
    cache = pc.PagedCache(k, v, *sc, None, BF)
    q = torch.randn(1, 16, 1, D, generator=g, device=DEV).to(BF)
    out = pc.paged_decode(q, cache, i32([far]), i32([1234]), 0.06)
    assert torch.equal(out, pc.paged_decode(q, small, i32([list(range(20))]), i32([1234]), 0.06))
    x = torch.randn(5, Hk, D, generator=g, device=DEV).to(BF)
    pc.paged_write(cache, x, x, i32([far]), i32([1234]), cu_new=i32([0, 5]))
    pc.paged_write(small, x, x, i32([list(range(20))]), i32([1234]), cu_new=i32([0, 5]))
    assert torch.equal(k[P - 20:], small.k_pages) and torch.equal(sc[1][P - 20:], small.v_scale)
    assert (k[:P - 20] == 0).all()


def test_selected_pages(hip_lib):
    """The selector's lists over a cache in four bits: pages by the keys as they were given."""
    g = gen(16)
    lens = [64 * 30, 64 * 12 + 5]
    table, P = tables(lens, g)
    cache = pc.PagedCache.empty(P, 2, 128, BF, DEV, e2m1=True)
    wide = pc.PagedCache.empty(P, 2, 128, BF, DEV)
    T = sum(lens)
    k, v = (torch.randn(T, 2, 128, generator=g, device=DEV).to(BF) for _ in range(2))
    cu = i32([0, lens[0], T])
    for c in (cache, wide):
        pc.paged_write(c, k, v, table, i32([0, 0]), cu_new=cu)
    q = torch.randn(2, 14, 1, 128, generator=g, device=DEV).to(BF)
    a = pc.paged_select(q, cache, table, i32(lens), 0.09, 6, 12, tau=0.05)
    b = pc.paged_select(q, wide, table, i32(lens), 0.09, 6, 12, tau=0.05)
    assert torch.equal(a.kv_idx, b.kv_idx) and torch.equal(a.counts, b.counts)
    check_decode(q, cache, table, lens, 0.09, kv_idx=a.kv_idx, counts=a.counts)


def test_decode_step_in_a_graph(hip_lib):
    """Turn, write, attend: captured once, replayed as the sequences grow."""
    g = gen(17)
    B, H, Hk, D = 3, 8, 2, 128
    rot = ro.Rotary.make(D, DEV)
    lens = i32([0, 62, 500])
    table, P = tables([80, 140, 580], g)
    qkv = torch.randn(B, H + 2 * Hk, D, generator=g, device=DEV).to(BF)
    caches = [filled(gen(18), P, Hk, D, BF) for _ in range(2)]
    for c in caches:
        pc.paged_write(c, *(torch.randn(500, Hk, D, generator=gen(19), device=DEV).to(BF) for _ in "kv"), table,
                       i32([0, 0, 0]), cu_new=i32([0, 0, 0, 500]))

    def step(cache):
        q = ro.rotary(rot, lens, qkv[:, :H])
        pc.paged_write(cache, qkv[:, H:H + Hk], qkv[:, H + Hk:], table, lens, rotary=rot)
        lens.add_(1)
        return pc.paged_decode(q.unsqueeze(2), cache, table, lens, 0.09)
    warm = lens.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(filled(gen(1), P, Hk, D, BF))
    torch.cuda.current_stream().wait_stream(side)
    lens.copy_(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    lens.copy_(warm)
    for i in range(6):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=DEV))
        now = lens.clone()
        want = step(caches[1])
        lens.copy_(now)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
        assert torch.equal(bits(caches[0].k_pages), bits(caches[1].k_pages))


def test_refusals(hip_lib):
    P, Hk, D = 2, 1, 64
    pages = torch.zeros(P, Hk, 64, D // 2, dtype=torch.uint8, device=DEV)
    sc = torch.zeros(P, Hk, D // 32, 64, dtype=torch.uint8, device=DEV)
    pc.PagedCache(pages, pages, sc, sc, None, BF)
    for bad in (lambda: pc.PagedCache(pages, pages, sc, sc), lambda: pc.PagedCache(pages, pages, None, None, None, BF),
                lambda: pc.PagedCache(pages, pages, sc[:, :, 0], sc[:, :, 0], None, BF),
                lambda: pc.PagedCache(pages[..., :16], pages[..., :16], sc, sc, None, BF),
                lambda: pc.PagedCache(pages, pages.view(torch.float8_e4m3fn), sc, sc, None, BF),
                lambda: pc.PagedCache.empty(2, 1, 64, BF, DEV, e4m3=True, e2m1=True)):
        with pytest.raises(AssertionError):
            bad()
    cache = pc.PagedCache.empty(P, Hk, D, BF, DEV, e2m1=True)
    k = torch.zeros(1, 1, D, dtype=BF, device=DEV)
    rot = ro.Rotary.make(128, DEV)
    for kw in (dict(rotary=rot), dict(positions=i32([0])), dict(rotary=ro.Rotary.make(64, DEV), positions=i32([0, 1]))):
        with pytest.raises(AssertionError):
            pc.paged_write(cache, k, k, i32([[0]]), i32([0]), **kw)
