"""Attention weights followed over a paged cache, and eviction by them, against 64-bit references on
the same inputs; and the serving operators one behind the other."""

import math

import pytest
import torch

import paged_cache as pc
import rotary as ro
import test_gpu_paged_cache as wide
import test_gpu_paged_e2m1 as four
from test_gpu_paged_cache import bits, gen, i32, tables

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, FH = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def filled(g, P, Hk, D, dtype, kind, interleaved=False):
    if kind == "e2m1":
        return four.filled(g, P, Hk, D, dtype, interleaved)
    return wide.filled(g, P, Hk, D, dtype, kind == "e4m3", interleaved)


def values(cache, name):
    return four.cache_values(cache, name) if cache.k_pages.dtype == torch.uint8 else wide.cache_values(cache, name)


# ---- weights ------------------------------------------------------------------------------------

def weights_ref(q, cache, table, lens, scale, kv_idx=None, counts=None):
    """[B, Hk, 64 * max_pages] fp64: what each token's weights add up to."""
    B, H, _, D = q.shape
    P, Hk, NB = cache.k_pages.shape[0], cache.k_pages.shape[1], table.shape[1]
    kc = values(cache, "k").to(q.dtype).double()
    out = torch.zeros(B, Hk, 64 * NB, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = min(max(lens[b], 0), 64 * NB)
        for h in range(Hk):
            blocks = range(NB) if kv_idx is None else kv_idx[b, h, :kv_idx.shape[2] if counts is None else
                                                            max(int(counts[b, h]), 0)].tolist()
            blocks = [j for j in blocks if 0 <= j < NB and 64 * j < n and 0 <= int(table[b, j]) < P]
            if not blocks:
                continue
            at = torch.tensor(blocks, device=DEV)
            tokens = (at.view(-1, 1) * 64 + torch.arange(64, device=DEV)).flatten()
            k = kc[table[b][at].long(), h].flatten(0, 1)[tokens < n]
            p = torch.softmax((q[b, h * (H // Hk):(h + 1) * (H // Hk), 0].double() @ k.T) * scale, -1)
            out[b, h, tokens[tokens < n]] += p.sum(0)
    return out


def check_weights(q, cache, table, lens, scale, start, **lists):
    """Weights of scores of ten or so: fp32 moves one by less than 1e-5 of itself, and the sum over the
    heads and with what was there rounds by 2^-24 of the result a time."""
    B, H, _, D = q.shape
    mass = start.clone()
    out = pc.paged_decode(q, cache, table, i32(lens), scale, mass=mass, **lists)
    assert torch.equal(out, pc.paged_decode(q, cache, table, i32(lens), scale, **lists))
    W = 64 * table.shape[1]
    want = weights_ref(q, cache, table, lens, scale, **lists)
    off = (mass[..., :W].double() - start[..., :W].double() - want).abs()
    assert (off <= 2e-5 * want + (H + 1) * 2.0 ** -24 * (start[..., :W].double().abs() + want)).all(), off.max()
    same = want == 0
    assert torch.equal(mass[..., :W][same], start[..., :W][same])
    assert torch.equal(mass[..., W:], start[..., W:])
    return mass


SHAPES = [(8, 8, 64, BF, "model"), (8, 2, 64, FH, "e4m3"), (28, 4, 128, BF, "model"), (34, 2, 128, FH, "e2m1"),
          (28, 4, 128, BF, "e4m3"), (16, 2, 256, BF, "model"), (9, 1, 256, FH, "e2m1"), (40, 8, 128, BF, "e2m1"),
          (7, 1, 64, BF, "e2m1")]


def poison(cache, table, lens):
    """NaN in every slot that holds no token of a sequence."""
    if cache.k_pages.dtype == torch.uint8:
        return four.poison(cache, table, lens)
    P = cache.k_pages.shape[0]
    dead = torch.ones(P, 64, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        for j in range((n + 63) // 64):
            dead[table[b, j], : n - 64 * j] = False
    for t in (cache.k_pages, cache.v_pages):
        t.copy_(t.float().masked_fill(dead.view(P, 1, 64, 1), NAN))


@pytest.mark.parametrize("lens", [[1], [0, 31, 32, 33, 63, 64, 65], [511, 0, 1000, 2], [4097], [130, 0, 256, 1] * 33])
@pytest.mark.parametrize("H,Hk,D,dtype,kind", SHAPES)
def test_weights(hip_lib, lens, H, Hk, D, dtype, kind):
    print(f"[case] weights {lens[:7]} H={H}/{Hk} D={D} {dtype} {kind}", flush=True)
    g = gen(D + H + len(lens))
    table, P = tables(lens, g)
    cache = filled(g, P, Hk, D, dtype, kind, interleaved=H == 28)
    poison(cache, table, lens)
    q = torch.randn(len(lens), 1, H, D, generator=g, device=DEV).to(dtype).transpose(1, 2)
    start = torch.rand(len(lens), Hk, 64 * table.shape[1] + 64, generator=g, device=DEV)
    check_weights(q, cache, table, lens, D ** -0.5, start)


@pytest.mark.parametrize("H,Hk,D,dtype,kind", SHAPES)
def test_weights_of_listed_pages(hip_lib, H, Hk, D, dtype, kind):
    g = gen(D + H + 2)
    lens = [64 * 40 - 5, 3, 64 * 9]
    table, P = tables(lens, g, width=41)
    cache = filled(g, P, Hk, D, dtype, kind)
    q = torch.randn(3, H, 1, D, generator=g, device=DEV).to(dtype)
    start = torch.rand(Hk, 3, 64 * 41, generator=g, device=DEV).transpose(0, 1)
    for slots in (1, 7, 60):
        order = torch.rand(3, Hk, 41, generator=g, device=DEV).argsort(-1)[..., :slots]
        idx = torch.full((3, Hk, slots), 41, dtype=torch.int32, device=DEV)
        idx[..., :order.shape[-1]] = order.to(torch.int32)
        idx[0, 0, 0] = -7
        counts = torch.randint(-1, slots + 1, (3, Hk), generator=g, device=DEV, dtype=torch.int32)
        check_weights(q, cache, table, lens, D ** -0.5, start, kv_idx=idx)
        check_weights(q, cache, table, lens, D ** -0.5, start, kv_idx=idx, counts=counts)


@pytest.mark.parametrize("kind", ["model", "e4m3", "e2m1"])
def test_weights_absent_pages_and_wide_tables(hip_lib, kind):
    g = gen(21)
    cache = filled(g, 40, 2, 128, BF, kind)
    q = torch.randn(4, 8, 1, 128, generator=g, device=DEV).to(BF)
    for width in (4, 100, 20000):
        table = torch.full((4, width), -1, dtype=torch.int32, device=DEV)
        table[:, :4] = i32([[0, -1, 47, 2], [5, 1, 6, -9], [-1, -1, -1, -1], [3, 4, 0, 1]])
        start = torch.rand(4, 2, 64 * width, generator=g, device=DEV)
        check_weights(q, cache, table, [256, 90, 200, 250], 0.09, start)
        check_weights(q, cache, table, [0, -5, 200, 1], 0.09, start)


@pytest.mark.parametrize("H,Hk,D,dtype,kind", [(8, 2, 64, BF, "model"), (34, 2, 128, FH, "e2m1"), (9, 1, 256, FH, "e2m1"),
                                               (16, 2, 128, BF, "e4m3"), (40, 8, 128, BF, "e2m1")])
def test_weights_of_several_live_tiles(hip_lib, H, Hk, D, dtype, kind):
    """Wide tables and lists, where a workgroup adds the weights of several runs of 1024 tokens, in rows
    that fill some of them, one or none."""
    print(f"[case] live tiles H={H}/{Hk} D={D} {dtype} {kind}", flush=True)
    g = gen(H + D)
    lens, width = [9001, 1025, 5120, 0, 6200, 1024], 20000
    B = len(lens)
    tiles = (width + 15) // 16 * Hk * B
    assert tiles > 2 * 1024                                  # a workgroup has three at least
    table, P = tables(lens, g, width=width)
    cache = filled(g, P, Hk, D, dtype, kind)
    poison(cache, table, lens)
    q = torch.randn(B, H, 1, D, generator=g, device=DEV).to(dtype)
    start = torch.rand(B, Hk, 64 * width, generator=g, device=DEV)
    check_weights(q, cache, table, lens, D ** -0.5, start)
    slots = 4096
    for counts in (None, torch.randint(17, 160, (B, Hk), generator=g, device=DEV, dtype=torch.int32)):
        idx = torch.full((B, Hk, slots), width, dtype=torch.int32, device=DEV)
        for b in range(B):
            n = (lens[b] + 63) // 64
            for h in range(Hk):                              # pages in any order, some that are none between
                order = torch.randperm(n + 20, generator=g, device=DEV)
                idx[b, h, :n + 20] = torch.where(order < n, order, width + 3).to(torch.int32)
        check_weights(q, cache, table, lens, D ** -0.5, start, kv_idx=idx, counts=counts)


def test_weights_of_nan_and_infinite_scores(hip_lib):
    """A NaN score makes its KV head's row NaN up to the length, and nothing past it."""
    g = gen(22)
    table, P = tables([100, 100], g, width=3)
    cache = filled(g, P, 2, 64, BF, "model")
    q = torch.randn(2, 4, 1, 64, generator=g, device=DEV).to(BF)
    cache.k_pages[table[0, 1].long(), 1, 9] = NAN
    mass = torch.ones(2, 2, 192, device=DEV)
    pc.paged_decode(q, cache, table, i32([100, 100]), 0.1, mass=mass)
    nan = torch.zeros_like(mass, dtype=torch.bool)
    nan[0, 1, :100] = True
    assert torch.equal(mass.isnan(), nan) and (mass[0, 1, 100:] == 1).all()
    # all scores -infinity: no weight anywhere
    cache.k_pages[:] = -INF
    mass = torch.ones(2, 2, 192, device=DEV)
    out = pc.paged_decode(torch.ones_like(q), cache, table, i32([100, 100]), 0.1, mass=mass)
    assert (out == 0).all() and (mass == 1).all()


def test_weights_repeat_themselves(hip_lib):
    g = gen(23)
    lens = [5000, 700, 64]
    table, P = tables(lens, g)
    cache = filled(g, P, 4, 128, BF, "e2m1")
    q = torch.randn(3, 28, 1, 128, generator=g, device=DEV).to(BF)
    sums = [torch.zeros(3, 4, 64 * table.shape[1], device=DEV) for _ in range(3)]
    for m in sums:
        for _ in range(3):
            pc.paged_decode(q, cache, table, i32(lens), 0.09, mass=m)
    assert torch.equal(sums[0], sums[1]) and torch.equal(sums[0], sums[2])
    total = sums[0].double().sum(-1)
    assert ((total - 3 * 7).abs() < 1e-3).all()                  # three steps of seven heads' unit weight


# ---- eviction -----------------------------------------------------------------------------------

def evict_ref(mass, table, lens, keep, recent, first, P):
    """Kept tokens by the definition: lists [B][Hk]."""
    rows, out = table.tolist(), []
    for b in range(mass.shape[0]):
        n = min(max(lens[b], 0), 64 * table.shape[1])
        have = [i for i in range(n) if 0 <= rows[b][i // 64] < P]
        out.append([])
        for h in range(mass.shape[1]):
            m = mass[b, h].tolist()
            rank = sorted(have, key=lambda i: (not (i < first or i >= n - recent), not math.isnan(m[i]),
                                               0 if math.isnan(m[i]) else -m[i], i))
            out[b].append(sorted(rank[:keep]))
    return out


def check_evict(cache, mass, table, lens, keep, recent, first, g, spare=0):
    """The call against the definition, bit for bit."""
    B, Hk, P = table.shape[0], cache.k_pages.shape[1], cache.k_pages.shape[0]
    used = set(table.flatten().tolist())
    fresh = [p for p in range(P) if p not in used]
    new_pages = (keep + 63) // 64 + spare
    assert len(fresh) >= B * new_pages
    order = torch.randperm(len(fresh), generator=g, device=DEV).tolist()
    new_table = i32([[fresh[order[b * new_pages + j]] for j in range(new_pages)] for b in range(B)])
    names = [n for n in ("k_pages", "v_pages", "k_scale", "v_scale", "planes") if getattr(cache, n) is not None]
    want = {n: getattr(cache, n).clone() for n in names}
    keys = values(cache, "k")
    kept = evict_ref(mass, table, lens, keep, recent, first, P)
    start = mass.clone()
    r = pc.paged_evict(cache, mass, table, i32(lens), new_table, keep, recent=recent, first=first)
    none = 64 * table.shape[1]
    for b in range(B):
        count = len(kept[b][0])
        assert int(r.seq_lens[b]) == count
        for h in range(Hk):
            assert r.kept[b, h].tolist() == kept[b][h] + [none] * (keep - count)
            if not count:
                assert (r.mass[b, h] == 0).all()
                continue
            tok, to = torch.tensor(kept[b][h], device=DEV), torch.arange(count, device=DEV)
            src, dst = table[b].long()[tok // 64], new_table[b].long()[to // 64]
            for n in names[:-1] if "planes" in names else names:
                if "scale" in n and cache.k_pages.dtype == torch.uint8:
                    want[n][dst, h, :, to % 64] = getattr(cache, n)[src, h, :, tok % 64]
                else:
                    bits_to, bits_from = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
                                          for t in (want[n], getattr(cache, n)))
                    bits_to[dst, h, to % 64] = bits_from[src, h, tok % 64]
            assert torch.equal(r.mass[b, h, :count].nan_to_num(nan=-1.0), start[b, h, tok].nan_to_num(nan=-1.0))
            assert (r.mass[b, h, count:] == 0).all()
            for j in range((count + 63) // 64 if "planes" in names else 0):
                x = keys[src, h, tok % 64][64 * j:64 * j + 64]
                both = torch.stack([torch.nan_to_num(x, nan=-INF).amax(0) if x.isnan().any() else x.amax(0),
                                    torch.nan_to_num(x, nan=INF).amin(0) if x.isnan().any() else x.amin(0)])
                want["planes"][new_table[b, j].long(), h] = both.to(cache.dtype)
    for n in names:
        # of zeros of either sign a summary may hold either: they are equal
        same = torch.equal if n == "planes" else lambda a, b: torch.equal(bits(a), bits(b))
        assert same(getattr(cache, n), want[n]), n
    assert torch.equal(bits(mass), bits(start))
    return r, new_table


@pytest.mark.parametrize("lens,keep,recent,first", [([1], 1, 0, 0), ([64, 65, 0, 63], 64, 0, 0), ([200, 7, 130], 100, 30, 4),
                                                    ([1000, 300], 65, 65, 0), ([1000, 2], 1, 0, 1), ([5000], 777, 50, 0),
                                                    ([4100, 4096], 3000, 0, 64), ([90], 128, 20, 20)])
@pytest.mark.parametrize("Hk,D,dtype,kind", [(4, 128, BF, "model"), (2, 64, FH, "e4m3"), (3, 256, BF, "e2m1"),
                                             (1, 64, BF, "e2m1"), (2, 256, FH, "model"), (2, 128, FH, "e2m1")])
def test_evict(hip_lib, lens, keep, recent, first, Hk, D, dtype, kind):
    print(f"[case] evict {lens} keep={keep} {recent} {first} Hk={Hk} D={D} {dtype} {kind}", flush=True)
    g = gen(D + Hk + keep)
    table, P = tables(lens, g, spare=2 + len(lens) * ((keep + 63) // 64 + 1))
    cache = filled(g, P, Hk, D, dtype, kind, interleaved=Hk == 4)
    mass = torch.exp(3 * torch.randn(len(lens), Hk, 64 * table.shape[1], generator=g, device=DEV))
    check_evict(cache, mass, table, lens, keep, recent, first, g, spare=len(lens) % 2)


def test_evict_ties_and_special_weights(hip_lib):
    """Equal weights stay by the lower token; NaN before numbers, zeros of either sign alike, infinities,
    subnormal and negative weights in their order."""
    g = gen(31)
    lens = [700, 700, 700, 700, 700, 700]
    table, P = tables(lens, g, spare=6 * 11 + 2)
    mass = torch.ones(6, 2, 64 * 11, device=DEV)
    mass[1] = torch.randint(0, 3, (2, 704), generator=g, device=DEV).float()
    mass[2] = torch.where(torch.rand(2, 704, generator=g, device=DEV) < 0.5, 0.0, -0.0)
    mass[3] = torch.tensor([NAN, INF, -INF, 0.0, -0.0, 1e-42, -1e-42, 1.0, -1.0, 3e38], device=DEV)[
        torch.randint(0, 10, (2, 704), generator=g, device=DEV)]
    mass[4] = NAN
    mass[5] = 1.0 + torch.randint(0, 5, (2, 704), generator=g, device=DEV) * 2.0 ** -23
    for keep, recent, first in ((1, 0, 0), (64, 3, 5), (300, 0, 0), (500, 499, 1), (699, 1, 0), (333, 111, 222)):
        cache = filled(gen(32), P, 2, 64, BF, "e4m3")
        check_evict(cache, mass, table, lens, keep, recent, first, g)


def test_evict_absent_pages(hip_lib):
    """Tokens of absent pages do not stay, even where they are among the newest."""
    g = gen(33)
    for kind in ("model", "e2m1"):
        cache = filled(g, 30, 2, 64, FH, kind)
        table = i32([[0, -1, 3, 99], [4, 5, -1, -1], [-1, -2, 30, 31], [6, 7, 8, 9]])
        mass = torch.rand(4, 2, 256, generator=g, device=DEV)
        for lens in ([256, 256, 256, 256], [200, 70, 1, 0], [-4, 1 << 30, 9, 129]):
            check_evict(cache, mass, table, lens, 100, 40, 3, g)


def test_evict_into_absent_pages(hip_lib):
    """Tokens without a page to go to are left out of it; the rest arrive."""
    g = gen(34)
    cache = filled(g, 12, 1, 64, BF, "model")
    table, before = i32([[0, 1, 2, 3]]), None
    before = {n: getattr(cache, n).clone() for n in ("k_pages", "v_pages", "planes")}
    mass = torch.rand(1, 1, 256, generator=g, device=DEV)
    r = pc.paged_evict(cache, mass, table, i32([256]), i32([[7, -1, 12, 9]]), 200)
    tok = r.kept[0, 0].long()
    assert int(r.seq_lens[0]) == 200
    for n in ("k_pages", "v_pages"):
        want = before[n]
        want[7, 0] = want[tok[:64] // 64, 0, tok[:64] % 64]
        want[9, 0, :8] = want[tok[192:] // 64, 0, tok[192:] % 64]
        assert torch.equal(getattr(cache, n), want)


def test_evict_long_rows(hip_lib):
    """Rows of more tokens than a workgroup's threads hold at once, nearly all weights alike."""
    g = gen(35)
    lens = [100000, 70001]
    held = [(n + 63) // 64 for n in lens]
    keep = 9000
    P = sum(held) + 2 * ((keep + 63) // 64)
    table = torch.full((2, max(held)), -1, dtype=torch.int32, device=DEV)
    table[0, :held[0]] = torch.arange(held[0])
    table[1, :held[1]] = torch.arange(held[0], sum(held))
    new_table = torch.arange(sum(held), P, device=DEV, dtype=torch.int32).view(2, -1)
    cache = filled(g, P, 2, 64, BF, "e2m1")
    W = 64 * max(held)
    for mass in (torch.rand(2, 2, W, generator=g, device=DEV), torch.randint(0, 40, (2, 2, W), generator=g, device=DEV).float(),
                 1 + 2.0 ** -23 * torch.randint(0, 9, (2, 2, W), generator=g, device=DEV)):
        r = pc.paged_evict(cache, mass, table, i32(lens), new_table, keep, recent=500, first=4)
        for b in range(2):
            order = mass[b, :, :lens[b]].clone()
            order[:, :4], order[:, lens[b] - 500:] = INF, INF
            want = order.sort(dim=-1, descending=True, stable=True)[1][:, :keep].sort(-1)[0]
            assert torch.equal(r.kept[b].long(), want)
            assert torch.equal(r.mass[b, :, :keep], mass[b].gather(-1, want))
            for h in range(2):
                t = want[h]
                to = torch.arange(keep, device=DEV)
                src, dst = table[b].long()[t // 64], new_table[b].long()[to // 64]
                assert torch.equal(cache.k_pages[dst, h, to % 64], cache.k_pages[src, h, t % 64])
                assert torch.equal(cache.v_scale[dst, h, :, to % 64], cache.v_scale[src, h, :, t % 64])


def pick_ref(row, tokens, n, keep, recent, first):
    """The tokens of one row that stay: `tokens` [n] true where there is a page."""
    i = torch.arange(n, device=DEV)
    sure = (i < first) | (i >= n - recent)
    x = row[:n] + 0.0
    # a rank: those that stay in any case, NaN, then by weight; the stable sort keeps ties in order
    x = torch.where(sure, INF, torch.where(x.isnan(), INF, x))
    order = x.sort(descending=True, stable=True)[1]
    cls = torch.where(sure, 0, torch.where(row[:n].isnan(), 1, 2))
    cls = torch.where(tokens, cls, 3)
    order = order[cls[order].sort(stable=True)[1]]
    return order[:min(keep, int(tokens.sum()))].sort()[0]


@pytest.mark.parametrize("width,B,Hk", [(129, 2, 3), (260, 2, 3), (520, 3, 2), (260, 11, 6), (520, 11, 6)])
def test_evict_rows_of_many_pages(hip_lib, width, B, Hk):
    """Few rows of many pages are picked by several workgroups each, many by one: cuts at the ends of
    their parts, first and newest tokens over several of them, absent pages, ties, NaN."""
    print(f"[case] rows of {width} pages, {B} x {Hk}", flush=True)
    g = gen(width + B)
    W = 64 * width
    cache = filled(g, 400, Hk, 64, BF, "e4m3")
    lens = [[W, 4097], [4096, 8192], [W - 1, 8193], [0, 1], [63, -3]]
    special = torch.tensor([NAN, INF, -INF, 0.0, -0.0, 1e-42, -1e-42, 1.0, -1.0, 3e38], device=DEV)

    def masses():
        yield torch.exp(3 * torch.randn(B, Hk, W, generator=g, device=DEV))
        yield torch.zeros(B, Hk, W, device=DEV)
        yield torch.randint(0, 3, (B, Hk, W), generator=g, device=DEV).float()
        yield special[torch.randint(0, 10, (B, Hk, W), generator=g, device=DEV)]
        yield torch.where(torch.rand(B, Hk, W, generator=g, device=DEV) < 0.3, NAN, 1.0)
        yield 1 + 2.0 ** -23 * torch.randint(0, 9, (B, Hk, W), generator=g, device=DEV)
        yield torch.rand(B, Hk, W, generator=g, device=DEV)

    for i, mass in enumerate(masses()):
        pages = torch.randint(0, 300, (B, width), generator=g, device=DEV, dtype=torch.int32)
        if i % 2:
            pages = torch.where(torch.rand(B, width, generator=g, device=DEV) < 0.2, -1, pages)
        lengths = [lens[i % 5][b % 2] for b in range(B)]
        for keep, recent, first in ((1, 0, 0), (200, 30, 4), (5000, 4500, 300), (5000, 0, 5000), (6000, 0, 0), (W, 0, 0)):
            new_table = torch.full((B, (keep + 63) // 64), -1, dtype=torch.int32, device=DEV)
            r = pc.paged_evict(cache, mass, pages, i32(lengths), new_table, keep, recent=recent, first=first)
            for b in {0, 1, B - 1}:
                n = min(max(lengths[b], 0), W)
                there = (pages[b] >= 0).repeat_interleave(64)[:n]
                want = [pick_ref(mass[b, h], there, n, keep, recent, first) for h in range(Hk)]
                assert int(r.seq_lens[b]) == len(want[0])
                for h in range(Hk):
                    assert torch.equal(r.kept[b, h, :len(want[h])].long(), want[h])
                    assert (r.kept[b, h, len(want[h]):] == W).all()


@pytest.mark.parametrize("width,B,Hk", [(20, 2, 2), (100, 1, 3), (500, 40, 2), (900, 2, 3), (2100, 8, 8)])
def test_evict_weights_that_agree(hip_lib, width, B, Hk):
    """Rows most of whose weights were never added to, or lie within one bin or at a few values in it, in
    every form of the pick: cuts among the zeros, among the others, and between the two."""
    print(f"[case] weights that agree, {width} pages, {B} x {Hk}", flush=True)
    g = gen(width)
    W = 64 * width
    cache = filled(g, 40, Hk, 64, BF, "e4m3")
    pages = torch.randint(0, 40, (B, width), generator=g, device=DEV, dtype=torch.int32)
    lens = [W - 7 * b if b % 3 < 2 else W // 2 + b for b in range(B)]
    some = torch.rand(B, Hk, W, generator=g, device=DEV)

    def masses():
        yield torch.where(some < 0.03, torch.exp(3 * torch.randn(B, Hk, W, generator=g, device=DEV)), 0.0)
        yield torch.where(some < 0.03, 1e-42, 0.0)                      # of the zeros' bin
        yield torch.where(torch.arange(W, device=DEV) % 1024 < 960, 0.0, some)      # whole wavefronts alike
        yield 1 + 0.2 * some
        yield torch.where(some < 0.6, 1.125, 1 + 0.2 * some)
        yield torch.where(torch.arange(W, device=DEV) < W // 2, 2.0, 2.25).expand(B, Hk, W).contiguous()
    for mass in masses():
        for keep, recent, first in ((W // 100, 0, 2), (W // 30, 5, 0), (W // 2, W // 8, 4)):
            new_table = torch.full((B, (keep + 63) // 64), -1, dtype=torch.int32, device=DEV)
            r = pc.paged_evict(cache, mass, pages, i32(lens), new_table, keep, recent=recent, first=first)
            for b in {0, 1 % B, 2 % B, B - 1}:
                there = torch.ones(lens[b], dtype=torch.bool, device=DEV)
                for h in range(Hk):
                    want = pick_ref(mass[b, h], there, lens[b], keep, recent, first)
                    assert int(r.seq_lens[b]) == len(want) and torch.equal(r.kept[b, h, :len(want)].long(), want)


def test_eviction_of_long_rows_replayed(hip_lib):
    """Captured at one set of lengths and weights, replayed at others beside another graph's replay."""
    g = gen(44)
    W, keep, B, Hk = 300, 700, 2, 2
    caches = [filled(gen(45), 40, Hk, 64, BF, "e4m3") for _ in range(2)]
    table = torch.randint(0, 20, (B, W), generator=g, device=DEV, dtype=torch.int32)
    new_table = torch.full((B, (keep + 63) // 64), -1, dtype=torch.int32, device=DEV)
    held = [(torch.rand(B, Hk, 64 * W, generator=g, device=DEV), i32([64 * W, 9000])) for _ in range(2)]
    pc.paged_evict(caches[0], *held[0][:1], table, held[0][1], new_table, keep, recent=9, first=3)
    torch.cuda.synchronize()
    graphs, results = [], []
    for cache, (mass, lens) in zip(caches, held):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(pc.paged_evict(cache, mass, table, lens, new_table, keep, recent=9, first=3))
        graphs.append(graph)
    for lengths in ([64 * W, 12345], [100, 4096], [0, 8193], [64 * W - 1, 1]):
        for mass, lens in held:
            mass.copy_(torch.randint(0, 50, mass.shape, generator=g, device=DEV))
            lens.copy_(i32(lengths))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for cache, (mass, lens), r in zip(caches, held, results):
            want = pc.paged_evict(cache, mass, table, lens, new_table, keep, recent=9, first=3)
            for got, x in ((r.kept, want.kept), (r.seq_lens, want.seq_lens), (r.mass, want.mass)):
                assert torch.equal(got, x)
            for b, n in enumerate(lengths):
                for h in range(Hk):
                    ref = pick_ref(mass[b, h], torch.ones(n, dtype=torch.bool, device=DEV), n, keep, 9, 3)
                    assert torch.equal(r.kept[b, h, :len(ref)].long(), ref)


def test_evict_of_a_shared_prefix(hip_lib):
    """Two sequences that share pages keep different tokens of them; the pages stay as they are."""
    g = gen(36)
    cache = filled(g, 20, 2, 128, BF, "e4m3")
    table = i32([[0, 1, 2, 3], [0, 1, 4, -1]])
    mass = torch.rand(2, 2, 256, generator=g, device=DEV)
    check_evict(cache, mass, table, [250, 190], 100, 10, 1, g)


def test_refusals(hip_lib):
    cache = filled(gen(37), 8, 2, 64, BF, "model")
    table, lens, mass = i32([[0, 1]]), i32([100]), torch.zeros(1, 2, 128, device=DEV)
    new = i32([[4, 5]])
    pc.paged_evict(cache, mass, table, lens, new, 64)
    q = torch.zeros(1, 4, 1, 64, device=DEV, dtype=BF)
    for bad in (dict(keep=0), dict(keep=129), dict(recent=65), dict(recent=-1), dict(first=-1), dict(recent=33, first=32),
                dict(new=new.long()), dict(new=new[:, :0]), dict(new=i32([[4], [5]])), dict(new=i32([[4, 0], [5, 0]]).T[:1]),
                dict(mass=mass[..., :127]), dict(mass=mass.half()), dict(mass=mass[:, :1]), dict(mass=mass[0]),
                dict(mass=torch.zeros(1, 2, 130, device=DEV)), dict(mass=torch.zeros(1, 2, 128)),
                dict(mass=torch.zeros(258, device=DEV)[2:].view(1, 2, 128)), dict(mass=mass.clone().requires_grad_()),
                dict(mass=torch.zeros(1, 2, 256, device=DEV)[..., ::2])):
        kw = dict(mass=mass, new=new, keep=64, recent=0, first=0)
        kw.update(bad)
        with pytest.raises(AssertionError):
            pc.paged_evict(cache, kw["mass"], table, lens, kw["new"], kw["keep"], recent=kw["recent"], first=kw["first"])
        if "mass" in bad:
            with pytest.raises(AssertionError):
                pc.paged_decode(q, cache, table, lens, 0.1, mass=kw["mass"])
    with pytest.raises(AssertionError, match="share"):
        pc.paged_decode(q, cache, table, lens, 0.1, mass=torch.zeros(1, 1, 128, device=DEV).expand(1, 2, 128))
    with pytest.raises(AssertionError, match="share"):
        pc.paged_decode(q.expand(2, 4, 1, 64), cache, table.expand(2, 2), i32([1, 1]), 0.1,
                        mass=torch.zeros(1024, device=DEV).as_strided((2, 2, 128), (64, 128, 1)))
    pages = torch.zeros(1, 2, 64, 64, device=DEV, dtype=BF).expand(8, 2, 64, 64)
    with pytest.raises(AssertionError, match="share"):
        pc.paged_evict(pc.PagedCache(pages, pages), mass, table, lens, new, 64)


# ---- all of it, as a server runs it -------------------------------------------------------------

@pytest.mark.parametrize("kind", ["model", "e4m3", "e2m1"])
def test_generation_within_a_budget(hip_lib, kind):
    """Prompts turned and written, tokens generated with their weights followed, the caches cut back, and
    on, against the same in 64 bits over lists of tokens."""
    g = gen(41)
    B, H, Hk, D, keep = 2, 6, 2, 64, 90
    rot = ro.Rotary.make(48, DEV, scaling="ntk", factor=2.0)
    prompt = [150, 100]
    P = 30
    cache = pc.PagedCache.empty(P, Hk, D, BF, DEV, e4m3=kind == "e4m3", e2m1=kind == "e2m1")
    table = i32([[0, 2, 4, 6], [1, 3, 5, 7]])
    lens, position = i32([0, 0]), i32(prompt)
    T = sum(prompt)
    qkv = torch.randn(T, H + 2 * Hk, D, generator=g, device=DEV).to(BF)
    cu = i32([0, prompt[0], T])
    pos = i32(list(range(prompt[0])) + list(range(prompt[1])))
    pc.paged_write(cache, qkv[:, H:H + Hk], qkv[:, H + Hk:], table, lens, cu_new=cu, rotary=rot)
    lens += i32(prompt)
    # the reference: per sequence and head the stored keys and values of the tokens it still has
    k, v = (t.double() for t in pc.paged_read(cache, table, lens, max(prompt)))
    turned = ro.rotary(rot, pos, qkv[:, H:H + Hk])
    if kind == "model":
        assert torch.equal(k[0, :, :150].transpose(0, 1), turned[:150].double())
    ref = [[(k[b, h, :prompt[b]], v[b, h, :prompt[b]], torch.zeros(prompt[b], dtype=torch.float64, device=DEV))
            for h in range(Hk)] for b in range(B)]
    mass = torch.zeros(B, Hk, 256, device=DEV)
    for step in range(45):
        qkv = torch.randn(B, H + 2 * Hk, D, generator=g, device=DEV).to(BF)
        q = ro.rotary(rot, position, qkv[:, :H])
        pc.paged_write(cache, qkv[:, H:H + Hk], qkv[:, H + Hk:], table, lens, rotary=rot, positions=position)
        lens += 1
        position += 1
        out = pc.paged_decode(q.unsqueeze(2), cache, table, lens, D ** -0.5, mass=mass)
        k, v = (t.double() for t in pc.paged_read(cache, table, lens, int(lens.max())))
        for b in range(B):
            n = int(lens[b])
            for h in range(Hk):
                kk, vv, w = ref[b][h]
                assert kk.shape[0] == n - 1 and torch.equal(k[b, h, :n - 1], kk)
                kk, vv = torch.cat([kk, k[b, h, n - 1:n]]), torch.cat([vv, v[b, h, n - 1:n]])
                p = torch.softmax(q[b, 3 * h:3 * h + 3].double() @ kk.T * D ** -0.5, -1)
                w = torch.cat([w, torch.zeros(1, dtype=torch.float64, device=DEV)]) + p.sum(0)
                ref[b][h] = kk, vv, w
                wide.check_close(out[b, 0, 3 * h:3 * h + 3], p @ vv, p @ vv.abs(), BF)
                assert (mass[b, h, :n].double() - w).abs().max() <= 1e-4
        if step in (14, 30):
            fresh = i32([[8, 10, 12, 14], [9, 11, 13, 15]]) if step == 14 else i32([[16, 18, 20, 22], [17, 19, 21, 23]])
            r = pc.paged_evict(cache, mass, table, lens, fresh, keep, recent=20, first=2)
            for b in range(B):
                for h in range(Hk):
                    kept = r.kept[b, h].long()
                    # by the weights as the kernels added them up (checked above)
                    assert kept.tolist() == evict_ref(mass, table, lens.tolist(), keep, 20, 2, P)[b][h]
                    ref[b][h] = tuple(t[kept] for t in ref[b][h])
            table, lens, mass = fresh, r.seq_lens, r.mass
            assert lens.tolist() == [keep, keep]
    # the summaries still bound what is cached: every page can be selected, and all of them are enough
    sel = pc.paged_select(q.unsqueeze(2), cache, table, lens, D ** -0.5, 4, 4)
    again = pc.paged_decode(q.unsqueeze(2), cache, table, lens, D ** -0.5, sel.kv_idx, sel.counts)
    for b in range(B):
        for h in range(Hk):
            kk, vv, _ = ref[b][h]
            p = torch.softmax(q[b, 3 * h:3 * h + 3].double() @ kk.T * D ** -0.5, -1)
            wide.check_close(again[b, 0, 3 * h:3 * h + 3], p @ vv, p @ vv.abs(), BF)


def test_step_and_eviction_in_graphs(hip_lib):
    """A decode step that follows weights, and an eviction, each captured once and replayed in turn with
    eager work between them."""
    g = gen(42)
    B, H, Hk, D, keep = 3, 8, 2, 128, 100
    start = [500, 120, 64]
    rot = ro.Rotary.make(D, DEV, interleaved=True)
    P = 40
    state = []
    for _ in range(2):
        cache = filled(gen(43), P, Hk, D, BF, "e2m1")
        table = torch.arange(30, device=DEV, dtype=torch.int32).view(3, 10)
        state.append(dict(cache=cache, table=table.clone(), lens=i32(start), pos=i32(start), qkv=torch.zeros(
            B, H + 2 * Hk, D, dtype=BF, device=DEV), mass=torch.zeros(B, Hk, 640, device=DEV), other=i32(
            [[30, 31], [32, 33], [34, 35]])))

    def step(s):
        q = ro.rotary(rot, s["pos"], s["qkv"][:, :H])
        pc.paged_write(s["cache"], s["qkv"][:, H:H + Hk], s["qkv"][:, H + Hk:], s["table"], s["lens"], rotary=rot,
                       positions=s["pos"])
        s["lens"] += 1
        s["pos"] += 1
        return pc.paged_decode(q.unsqueeze(2), s["cache"], s["table"], s["lens"], 0.09, mass=s["mass"])

    def evict(s):
        return pc.paged_evict(s["cache"], s["mass"], s["table"], s["lens"], s["other"], keep, recent=10)

    spare = dict(state[0], lens=state[0]["lens"].clone(), pos=state[0]["pos"].clone(), mass=state[0]["mass"].clone(),
                 cache=filled(gen(1), P, Hk, D, BF, "e2m1"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(spare), evict(spare)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    a, b = state
    stepped, evicted = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(stepped):
        out = step(a)
    with torch.cuda.graph(evicted):
        r = evict(a)
    for i in range(4):
        for s in state:
            s["qkv"].copy_(torch.randn(B, H + 2 * Hk, D, generator=gen(50 + i), device=DEV))
        torch.cuda.synchronize()
        stepped.replay()
        want = step(b)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(a["mass"], b["mass"]), i
        evicted.replay()
        w = evict(b)
        torch.cuda.synchronize()
        assert torch.equal(r.kept, w.kept) and torch.equal(r.seq_lens, w.seq_lens) and torch.equal(r.mass, w.mass)
        for n in ("k_pages", "v_pages", "k_scale", "v_scale", "planes"):
            assert torch.equal(bits(getattr(a["cache"], n)), bits(getattr(b["cache"], n))), (i, n)


def test_two_streams_at_once(hip_lib):
    """Two caches stepped on two streams: workspaces and results are each call's own."""
    g = gen(44)
    lens = [3000, 900]
    table, P = tables(lens, g)
    caches = [filled(gen(i), P, 4, 128, BF, "e2m1") for i in (1, 2)]
    q = torch.randn(2, 28, 1, 128, generator=g, device=DEV).to(BF)
    start = torch.rand(2, 4, 64 * table.shape[1], generator=g, device=DEV)
    want = []
    for c in caches:
        m = start.clone()
        want.append((pc.paged_decode(q, c, table, i32(lens), 0.09, mass=m), m))
    streams = [torch.cuda.Stream() for _ in caches]
    sums = [[start.clone() for _ in range(8)] for _ in caches]
    n = i32(lens)
    got = [[], []]
    torch.cuda.synchronize()
    for i in range(8):
        for j, (c, s) in enumerate(zip(caches, streams)):
            with torch.cuda.stream(s):
                got[j].append(pc.paged_decode(q, c, table, n, 0.09, mass=sums[j][i]))
    torch.cuda.synchronize()
    for j in range(2):
        for i in range(8):
            assert torch.equal(got[j][i], want[j][0]) and torch.equal(sums[j][i], want[j][1])
