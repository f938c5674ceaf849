"""Paged key-value cache: writing, reading back, page selection and decode attention against 64-bit
references on the same inputs."""

import math

import pytest
import torch

import _capi
import paged_cache as pc
import sparse_attention as sa
from block_attn import decode_attn

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, FH = torch.bfloat16, torch.float16
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def tables(lens, g, spare=2, width=None):
    """(block_table, pages): each sequence's pages scattered over the pool, -1 past them."""
    held = [(n + 63) // 64 for n in lens]
    P = sum(held) + spare
    order = torch.randperm(P, generator=g, device=DEV).tolist()
    width = width or max(max(held), 1)
    rows, at = [], 0
    for h in held:
        rows.append(order[at:at + h] + [-1] * (width - h))
        at += h
    return i32(rows), P


# ---- e4m3 by its definition ---------------------------------------------------------------------

def e4m3_ref(x, dtype):
    """(values of the codes, scale byte) of x [..., D] fp64: four significant bits, steps of 2^-9
    below 2^-6, ties to even; the scale the smallest power of two with max |x| <= 448 scale."""
    top = 61440.0 if dtype == FH else 1.875 * 2.0 ** 127
    x = x.clamp(-top, top)
    mx = torch.nan_to_num(x, nan=0.0).abs().amax(-1)
    e = [0 if m == 0 else max(math.frexp(m)[1] - 9 + (math.frexp(m)[0] > 0.875), -127)
         for m in mx.flatten().tolist()]
    e = torch.tensor(e, dtype=torch.float64, device=x.device).view(mx.shape)
    y = x * torch.exp2(-e).unsqueeze(-1)
    mag = y.abs().clamp(min=2.0 ** -6)
    step = torch.exp2(torch.frexp(mag)[1].double() - 4)
    return torch.round(y / step) * step, (e + 127).to(torch.uint8)


def cache_values(cache, name):
    """The pool of a cache as fp64 values [P, Hk, 64, D]."""
    x = getattr(cache, name + "_pages").double()
    scale = getattr(cache, name + "_scale")
    return x if scale is None else x * torch.exp2(scale.double() - 127).unsqueeze(-1)


def filled(g, P, Hk, D, dtype, e4m3, interleaved=False):
    """A cache of random pages."""
    if interleaved:       # K and V of a page side by side in one pool
        pool = torch.empty(P, 2, Hk, 64, D, dtype=torch.float8_e4m3fn if e4m3 else dtype, device=DEV)
        k, v = pool[:, 0], pool[:, 1]
        sc = [torch.empty(P, Hk, 64, dtype=torch.uint8, device=DEV) if e4m3 else None for _ in range(2)]
        cache = pc.PagedCache(k, v, *sc, torch.empty(P, Hk, 2, D, dtype=dtype, device=DEV), dtype)
    else:
        cache = pc.PagedCache.empty(P, Hk, D, dtype, DEV, e4m3=e4m3)
    for t in (cache.k_pages, cache.v_pages):
        x = torch.randn(P, Hk, 64, D, generator=g, device=DEV)
        t.copy_((x * 128).clamp(-448, 448) if e4m3 else x)
    if e4m3:
        for t in (cache.k_scale, cache.v_scale):
            t.copy_(torch.randint(118, 122, t.shape, generator=g, device=DEV))
    mid = torch.randn(P, Hk, D, generator=g, device=DEV)
    cache.planes.copy_(torch.stack([mid + 1.5, mid - 1.5], 2))
    return cache


# ---- write --------------------------------------------------------------------------------------

def written(cache, k, v, table, lens, new):
    """What the cache holds after the new tokens (bytes of its tensors), by loops."""
    e4m3 = cache.k_scale is not None
    out = {n: getattr(cache, n).clone() for n in ("k_pages", "v_pages", "k_scale", "v_scale", "planes")
           if getattr(cache, n) is not None}
    rows, P, at = table.tolist(), cache.k_pages.shape[0], 0
    for b, (n, m) in enumerate(zip(lens, new)):
        for i in range(m):
            pos = n + i
            page = rows[b][pos // 64] if pos // 64 < len(rows[b]) else -1
            if not 0 <= page < P:
                continue
            for name, x in (("k", k), ("v", v)):
                x = x[at + i]
                if e4m3:
                    val, byte = e4m3_ref(x.double(), cache.dtype)
                    out[name + "_scale"][page, :, pos % 64] = byte
                    x = val.to(torch.float8_e4m3fn)
                out[name + "_pages"][page, :, pos % 64] = x
            key, pl = k[at + i], out["planes"][page]
            if pos % 64 == 0:
                pl[:, 0], pl[:, 1] = -INF, INF
            pl[:, 0], pl[:, 1] = torch.fmax(pl[:, 0], key), torch.fmin(pl[:, 1], key)
        at += m
    return out


def bits(t):
    return t.contiguous().view(torch.uint8)


def check_written(cache, want):
    torch.cuda.synchronize()
    for name, t in want.items():
        assert torch.equal(bits(getattr(cache, name)), bits(t)), name


# Nothing new, one token, whole and part pages, a start inside a page, prompts over several pages
# with and without a cached prefix.
@pytest.mark.parametrize("lens,new", [([0], [1]), ([63], [1]), ([64], [1]), ([5, 0, 130], [0, 70, 1]),
                                      ([0, 1, 63, 64, 100], [64, 63, 2, 128, 300])])
@pytest.mark.parametrize("Hk,D,dtype,e4m3", [(4, 128, BF, True), (2, 64, FH, True), (1, 256, BF, True),
                                             (3, 256, FH, True), (8, 64, BF, False), (2, 128, FH, False)])
def test_write_ragged(hip_lib, lens, new, Hk, D, dtype, e4m3):
    print(f"[case] write {lens} {new} Hk={Hk} D={D} {dtype} {e4m3}", flush=True)
    g = gen(D + Hk)
    table, P = tables([a + b for a, b in zip(lens, new)], g)
    cache = filled(g, P, Hk, D, dtype, e4m3)
    T = sum(new)
    kv = torch.randn(T + 3, 2, Hk, D, generator=g, device=DEV)       # three rows of padding behind
    kv = (kv * torch.exp(2 * torch.randn(T + 3, 2, Hk, 1, generator=g, device=DEV))).to(dtype)
    k, v = kv[:, 0], kv[:, 1]
    want = written(cache, k, v, table, lens, new)
    cu = i32([sum(new[:i]) for i in range(len(new) + 1)])
    pc.paged_write(cache, k, v, table, i32(lens), cu_new=cu)
    check_written(cache, want)


@pytest.mark.parametrize("B", [1, 3, 300])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("dtype,e4m3", [(BF, True), (FH, False)])
def test_write_one_token_each(hip_lib, B, ragged, dtype, e4m3):
    """A decode step, by row or by ranges (more sequences than a workgroup has threads)."""
    g = gen(B)
    lens = [(17 * i) % 150 for i in range(B)]
    table, P = tables([n + 1 for n in lens], g)
    cache = filled(g, P, 2, 128, dtype, e4m3, interleaved=True)
    k, v = (torch.randn(B, 2, 128, generator=g, device=DEV).to(dtype) for _ in range(2))
    want = written(cache, k, v, table, lens, [1] * B)
    pc.paged_write(cache, k, v, table, i32(lens), cu_new=i32(list(range(B + 1))) if ragged else None)
    check_written(cache, want)


def test_write_special_values(hip_lib):
    """Zeros, subnormals, the largest values, infinities and NaN, each a token of its own."""
    for dtype, big in ((FH, 65504.0), (BF, 3.3895e38)):
        rows = [[0.0] * 64, [big] + [1.0] * 63, [-big] + [0.25] * 63, [INF, -INF] + [2.0] * 62,
                [NAN, 1.0, -448.0] + [0.5] * 61, [NAN] * 64, [6e-8] * 64, [6e-8, 1.2e-7] + [3e-5] * 62,
                [448.0] + [17.0] * 63, [449.0] + [17.0] * 63, [464.0, -9.5, 2.0 ** -9] + [1e-3] * 61]
        if dtype == BF:      # subnormal and the smallest scales
            rows += [[1e-40] * 64, [9.2e-41, 1.8e-40] + [0.0] * 62, [1.2e-38] + [1e-39] * 63]
        x = torch.tensor(rows, device=DEV).to(dtype).view(len(rows), 1, 64)
        cache = pc.PagedCache.empty(1, 1, 64, dtype, DEV, e4m3=True)
        pc.paged_write(cache, x, x, i32([[0]]), i32([0]), cu_new=i32([0, len(rows)]))
        val, byte = e4m3_ref(x.double(), dtype)
        for name in ("k", "v"):
            assert torch.equal(getattr(cache, name + "_scale")[0, 0, :len(rows)], byte[:, 0])
            got = getattr(cache, name + "_pages")[0, 0, :len(rows)].double()
            same = (got == val[:, 0]) | (got.isnan() & val[:, 0].isnan())
            assert same.all(), (dtype, (~same).nonzero().tolist())
        # reading back is exact in the model's dtype
        k, _ = pc.paged_read(cache, i32([[0]]), i32([len(rows)]), len(rows))
        want = (val * torch.exp2(byte.double() - 127).unsqueeze(-1))[:, 0]
        same = (k[0, 0].double() == want) | (k[0, 0].isnan() & want.isnan())
        assert same.all(), (dtype, (~same).nonzero().tolist())
        # NaN is passed over by the summary, infinities are in it
        assert torch.isposinf(cache.planes[0, 0, 0, 0]) and torch.isneginf(cache.planes[0, 0, 1, 1])


def test_write_leaves_out_what_has_no_page(hip_lib):
    """Tokens past the table, absent pages, negative lengths, offsets outside the tokens."""
    g = gen(1)
    cache = filled(g, 4, 2, 64, BF, True)
    k, v = (torch.randn(200, 2, 64, generator=g, device=DEV).to(BF) for _ in range(2))
    for table, lens, cu, new in [([[0, 1]], [100], [0, 200], [28]),             # 28 slots left
                                 ([[0, -1, 4, 2]], [0], [0, 200], [200]),       # two absent pages
                                 ([[0], [1]], [1 << 30, -5], [0, 3, 10], [0, 7]),
                                 ([[0], [1], [2]], [0, 0, 0], [-9, 4, 500, 3], [4, 64, 0])]:
        n = [max(x, 0) for x in lens]
        want = written(cache, k, v, i32(table), [min(x, 64 * len(table[0])) for x in n], new) \
            if cu[0] == 0 and cu[1] == 200 else None
        if cu[0] == -9:
            want = written(cache, k, v, i32(table), n, new)
        elif want is None:
            want = written(cache, k[3:], v[3:], i32(table), n, new)
        pc.paged_write(cache, k, v, i32(table), i32(lens), cu_new=i32(cu))
        check_written(cache, want)
    want = {"k_pages": cache.k_pages.clone(), "planes": cache.planes.clone()}
    pc.paged_write(cache, k[:0], v[:0], i32([[0]]), i32([0]), cu_new=i32([0, 0]))
    pc.paged_write(cache, k[:1], v[:1], i32([[0]]), i32([64]))                  # full table
    check_written(cache, want)


def test_planes_are_the_block_summary(hip_lib):
    """Token by token or at once, the planes of full pages are kernel 1's Quest planes."""
    g = gen(2)
    N, Hk, D = 192, 2, 128
    k = torch.randn(1, Hk, N, D, generator=g, device=DEV).to(BF)
    planes = sa.block_summary(k, _capi.MODE_QUEST).view(1, Hk, 3, 2, D)
    tok = k[0].transpose(0, 1)
    for steps in ([192], [1] * 192, [50, 30, 112]):
        cache = pc.PagedCache.empty(3, Hk, D, BF, DEV, e4m3=True)
        at = 0
        for n in steps:
            pc.paged_write(cache, tok[at:at + n], tok[at:at + n], i32([[2, 0, 1]]), i32([at]), cu_new=i32([0, n]))
            at += n
        assert torch.equal(cache.planes[[2, 0, 1]].transpose(0, 1), planes[0])


# ---- read ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("lens,n", [([1], 1), ([64], 64), ([0, 65, 200], 200), ([130, 7], 129), ([3], 300)])
@pytest.mark.parametrize("Hk,D,dtype,e4m3", [(4, 128, BF, True), (2, 64, FH, True), (1, 256, FH, True),
                                             (2, 256, BF, False)])
def test_read(hip_lib, lens, n, Hk, D, dtype, e4m3):
    g = gen(n + D)
    table, P = tables(lens, g)
    cache = filled(g, P, Hk, D, dtype, e4m3, interleaved=D == 64)
    out = torch.full((2, len(lens), n, Hk, D), NAN, dtype=dtype, device=DEV).transpose(2, 3)
    got = pc.paged_read(cache, table, i32(lens), n, out=(out[0], out[1]))
    fresh = pc.paged_read(cache, table, i32(lens), n)
    rows = table.tolist()
    for name, t, u in zip("kv", got, fresh):
        want = torch.zeros(len(lens), Hk, n, D, dtype=torch.float64, device=DEV)
        vals = cache_values(cache, name)
        for b, m in enumerate(lens):
            for i in range(min(m, n)):
                want[b, :, i] = vals[rows[b][i // 64], :, i % 64]
        assert torch.equal(t.double(), want) and torch.equal(u, t) and u.is_contiguous()


def test_read_absent_pages(hip_lib):
    cache = filled(gen(3), 3, 2, 64, BF, False)
    k, v = pc.paged_read(cache, i32([[1, 3, 2, -1]]), i32([1 << 20]), 256)
    for t, p in ((k, cache.k_pages), (v, cache.v_pages)):
        assert torch.equal(t[0, :, :64], p[1]) and torch.equal(t[0, :, 128:192], p[2])
        assert (t[0, :, 64:128] == 0).all() and (t[0, :, 192:] == 0).all()


# ---- select -------------------------------------------------------------------------------------

def select_ref(q, planes, table, lens, scale, k_base, k_slots, tau):
    """Lists, counts, sigma and flags by the definition, in fp64."""
    B, H, _, D = q.shape
    Hk, NB = planes.shape[1], table.shape[1]
    rows = table.tolist()
    lists = torch.full((B, Hk, k_slots), NB, dtype=torch.int32)
    counts = torch.zeros(B, Hk, dtype=torch.int32)
    sigma = torch.full((B, Hk), 2.0, dtype=torch.float64)
    flags = torch.zeros(B, Hk, dtype=torch.uint8)
    for b in range(B):
        nb = min((max(lens[b], 0) + 63) // 64, NB)
        for h in range(Hk):
            score = []
            for j in range(nb):
                if not 0 <= rows[b][j] < planes.shape[0]:
                    score.append(-INF)
                    continue
                hi, lo = planes[rows[b][j], h].double()
                x = q[b, h * (H // Hk):(h + 1) * (H // Hk), 0].double()
                score.append((torch.where(x >= 0, x * hi, x * lo)).sum(-1).max().item())
            rest = sorted(range(1, nb - 1), key=lambda j: (-score[j], j))
            keep, k = min(k_base, nb), k_base - 2
            if nb > k_base:
                s = [score[j] * scale for j in rest]
                with_cut = (s[k - 1] - s[k]) / max(s[0] - s[k], 1e-9)
                sigma[b, h] = min(max(with_cut, 0.0), 2.0)
                if sigma[b, h] < tau:
                    flags[b, h], keep = 1, min(k_slots, nb)
            kept = list(range(nb)) if nb <= keep else sorted([0, nb - 1] + rest[:keep - 2])
            lists[b, h, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
            counts[b, h] = keep
    return lists.to(DEV), counts.to(DEV), sigma.to(DEV), flags.to(DEV)


def check_select(q, cache, table, lens, scale, k_base, k_slots, tau):
    r = pc.paged_select(q, cache, table, i32(lens), scale, k_base, k_slots, tau=tau)
    want = select_ref(q, cache.planes, table, lens, scale, k_base, k_slots, tau)
    assert torch.equal(r.counts, want[1]) and torch.equal(r.uncertain, want[3])
    assert torch.equal(r.kv_idx, want[0])
    # rounded once to fp32 from fp64 scores
    assert ((r.sigma.double() - want[2]).abs() <= 2.0 ** -24 * want[2] + 1e-12).all()
    return r


@pytest.mark.parametrize("lens", [[0, 1, 64, 65, 128, 129], [320, 321, 383, 384, 385, 5000], [17000, 3]])
@pytest.mark.parametrize("H,Hk,D,dtype", [(8, 2, 128, BF), (4, 4, 64, FH), (34, 2, 128, FH), (16, 2, 256, BF),
                                          (7, 1, 64, BF), (40, 2, 256, FH)])
def test_select(hip_lib, lens, H, Hk, D, dtype):
    print(f"[case] select {lens} H={H}/{Hk} D={D} {dtype}", flush=True)
    g = gen(D + H + len(lens))
    table, P = tables(lens, g)
    cache = filled(g, P, Hk, D, dtype, False)
    q = torch.randn(len(lens), 1, H, D, generator=g, device=DEV).to(dtype).transpose(1, 2)
    for k_base, k_slots, tau in ((5, 10, 0.01), (3, 3, 0.0), (6, 9, 1e9), (300, 700, 0.02)):
        check_select(q, cache, table, lens, D ** -0.5, k_base, k_slots, tau)


def test_select_ties_take_the_lower_page(hip_lib):
    """Equal pages, pages of equal score by other keys, and a page that occurs twice."""
    cache = filled(gen(5), 40, 1, 64, BF, False)
    q = torch.ones(1, 2, 1, 64, device=DEV, dtype=BF)
    cache.planes[:] = 1.0
    cache.planes[3::4, :, :, 0], cache.planes[3::4, :, :, 1] = 1.5, 0.5       # the same sum
    cache.planes[9] += 1
    table = i32([list(range(39)) + [9]])
    table[0, 30] = 9
    for k_base, k_slots, tau in ((7, 14, 0.1), (7, 14, 0.0), (4, 38, 3.0), (39, 39, 0.0)):
        check_select(q, cache, table, [40 * 64], 0.125, k_base, k_slots, tau)


def test_select_special_scores(hip_lib):
    """Infinite planes, absent pages, scores of either sign of zero; NaN ranks first."""
    g = gen(6)
    cache = filled(g, 30, 2, 64, FH, False)
    cache.planes[4, 0, 0, 3] = INF
    cache.planes[5, :, :, :] = 0.0
    cache.planes[6, :, :, :] = -0.0
    q = torch.randn(1, 4, 1, 64, generator=g, device=DEV).abs().to(FH)
    table = i32([list(range(20)) + [-1, 30, 99] + list(range(20, 29))])
    check_select(q, cache, table, [32 * 64 - 5], 0.125, 12, 24, 1e-4)
    q.zero_()                                             # every score 0 (or 0 * inf)
    cache.planes[4, 0, 0, 3] = 1.0
    check_select(q, cache, table, [32 * 64 - 5], 0.125, 12, 24, 0.5)
    cache.planes[17, 1, 0, 0] = NAN
    r = pc.paged_select(q, cache, table, i32([32 * 64]), 0.125, 3, 3)
    assert r.kv_idx[0].tolist() == [[0, 1, 31], [0, 17, 31]]


def test_select_long_rows(hip_lib):
    """More pages than a workgroup holds at once, a table wider than the sequences."""
    g = gen(7)
    B, Hk, D, NB = 2, 2, 64, 20000
    planes = torch.randn(NB, Hk, D, generator=g, device=DEV)
    cache = pc.PagedCache(None, None, planes=torch.stack([planes + 1, planes - 1], 2).to(BF).contiguous())
    table = torch.stack([torch.randperm(NB, generator=g, device=DEV) for _ in range(B)]).int()
    q = torch.randn(B, 8, 1, D, generator=g, device=DEV).to(BF)
    lens = [NB * 64, 12345 * 64 + 1]
    r = pc.paged_select(q, cache, table, i32(lens), 0.125, 256, 512, tau=1e-3)
    for b in range(B):
        nb = (lens[b] + 63) // 64
        pl = cache.planes[table[b, :nb].long()].double()
        x = q[b, :, 0].double().view(Hk, 4, 1, D)
        s = torch.where(x >= 0, x * pl[:, :, 0].transpose(0, 1).unsqueeze(1),
                        x * pl[:, :, 1].transpose(0, 1).unsqueeze(1)).sum(-1).amax(1)
        s[:, 0] = s[:, -1] = INF
        for h in range(Hk):
            n = int(r.counts[b, h])
            order = s[h].sort(descending=True, stable=True)[1][:n].sort()[0]
            assert torch.equal(r.kv_idx[b, h, :n].long(), order) and (r.kv_idx[b, h, n:] == NB).all()


# ---- decode -------------------------------------------------------------------------------------

def decode_ref(q, cache, table, lens, scale, kv_idx=None, counts=None):
    """(out, sum of p |v|) [B, 1, H, D] in fp64."""
    B, H, _, D = q.shape
    Hk, P = cache.k_pages.shape[1], cache.k_pages.shape[0]
    kc, vc = cache_values(cache, "k"), cache_values(cache, "v")
    rows, NB = table.tolist(), table.shape[1]
    out = torch.zeros(2, B, 1, H, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = min(max(lens[b], 0), 64 * NB)
        for h in range(Hk):
            blocks = range((n + 63) // 64)
            if kv_idx is not None:
                m = kv_idx.shape[2] if counts is None else int(counts[b, h])
                blocks = [j for j in kv_idx[b, h, :max(m, 0)].tolist() if 0 <= j < (n + 63) // 64]
            blocks = [j for j in blocks if 0 <= rows[b][j] < P]
            if not blocks:
                continue
            at = torch.tensor(blocks, device=DEV)
            pages = table[b][at].long()
            live = ((at.view(-1, 1) * 64 + torch.arange(64, device=DEV)) < n).flatten()
            k, v = kc[pages, h].flatten(0, 1)[live], vc[pages, h].flatten(0, 1)[live]
            hs = slice(h * (H // Hk), (h + 1) * (H // Hk))
            p = torch.softmax((q[b, hs, 0].double() @ k.T) * scale, -1)
            out[0, b, 0, hs], out[1, b, 0, hs] = p @ v, p @ v.abs()
    return out[0], out[1]


def bound(ref, mass, dtype):
    """P and the output are rounded once each to the element format, by at most eps / 2 of the value
    (a weight below fp16's normal range by 2^-25 of the largest instead); e4m3 values are exact.
    fp32 scores and sums move a weight by less than 1e-5 of itself, and the normaliser with them."""
    u = torch.finfo(dtype).eps / 2
    return u * (mass + ref.abs()) + 2e-5 * mass + 1e-7


def check_close(out, ref, mass, dtype, times=1):
    off = ((out.double() - ref).abs() / (times * bound(ref, mass, dtype))).max().item()
    assert off <= 1.0, off


def check_decode(q, cache, table, lens, scale, **lists):
    out = pc.paged_decode(q, cache, table, i32(lens), scale, **lists)
    assert out.shape == (q.shape[0], 1, q.shape[1], q.shape[3]) and out.is_contiguous()
    ref, mass = decode_ref(q, cache, table, lens, scale, **lists)
    check_close(out, ref, mass, q.dtype)
    return out


SHAPES = [(8, 8, 64, BF, False), (8, 2, 64, FH, True), (28, 4, 128, BF, False), (34, 2, 128, FH, False),
          (28, 4, 128, BF, True), (34, 2, 128, FH, True), (16, 2, 256, BF, False), (9, 1, 256, FH, True),
          (16, 2, 256, BF, True), (4, 4, 64, BF, True)]


# Lengths around the step, the page and the splits, with slots without a sequence; slots past a
# length and pages of no sequence hold NaN.
@pytest.mark.parametrize("lens", [[1], [0, 31, 32, 33, 63, 64, 65], [511, 0, 1000, 2], [4097], [300] * 40,
                                  [130, 0, 256, 1] * 33])
@pytest.mark.parametrize("H,Hk,D,dtype,e4m3", SHAPES)
def test_decode(hip_lib, lens, H, Hk, D, dtype, e4m3):
    print(f"[case] paged decode {lens[:7]} H={H}/{Hk} D={D} {dtype} {e4m3}", flush=True)
    g = gen(D + H + len(lens))
    table, P = tables(lens, g)
    cache = filled(g, P, Hk, D, dtype, e4m3, interleaved=H == 28)
    dead = torch.ones(P, 64, dtype=torch.bool, device=DEV)
    for b, n in enumerate(lens):
        for j in range((n + 63) // 64):
            dead[table[b, j], : n - 64 * j] = False
    for t in (cache.k_pages, cache.v_pages):
        t.copy_(t.float().masked_fill(dead.view(P, 1, 64, 1), NAN))
    if e4m3:
        cache.v_scale.masked_fill_(dead.view(P, 1, 64), 255)
    q = torch.randn(len(lens), 1, H, D, generator=g, device=DEV).to(dtype).transpose(1, 2)
    out = check_decode(q, cache, table, lens, D ** -0.5)
    for b, n in enumerate(lens):
        assert n or (out[b] == 0).all()


# Lists with and without counts: shorter than the pages, padded in the middle, one page, none.
@pytest.mark.parametrize("H,Hk,D,dtype,e4m3", SHAPES)
def test_decode_listed(hip_lib, H, Hk, D, dtype, e4m3):
    g = gen(D + H)
    lens, slots = [1, 64, 700, 1500, 0, 4000], 21
    table, P = tables(lens, g)
    NB = table.shape[1]
    cache = filled(g, P, Hk, D, dtype, e4m3)
    q = torch.randn(len(lens), H, 1, D, generator=g, device=DEV).to(dtype)
    kv = torch.full((len(lens), Hk, slots), NB, dtype=torch.int32, device=DEV)
    counts = torch.zeros(len(lens), Hk, dtype=torch.int32, device=DEV)
    for b, n in enumerate(lens):
        nb = (n + 63) // 64
        for h in range(Hk):
            m = min(nb, 1 + (5 * b + 3 * h) % slots)
            kv[b, h, :m] = torch.randperm(nb, generator=g, device=DEV)[:m].sort()[0]
            counts[b, h] = m
    check_decode(q, cache, table, lens, D ** -0.5, kv_idx=kv, counts=counts)
    check_decode(q, cache, table, lens, D ** -0.5, kv_idx=kv)
    kv[:, :, 1] = -7                                      # no page of the sequence
    kv[:, :, 3] = 1 << 24
    check_decode(q, cache, table, lens, D ** -0.5, kv_idx=kv)
    counts.fill_(2)
    counts[3] = -1
    check_decode(q, cache, table, lens, -0.05, kv_idx=kv, counts=counts)
    counts.fill_(1 << 30)
    check_decode(q, cache, table, lens, D ** -0.5, kv_idx=kv, counts=counts.clamp(max=slots))
    a = pc.paged_decode(q, cache, table, i32(lens), 0.1, kv_idx=kv, counts=counts)
    assert torch.equal(a, pc.paged_decode(q, cache, table, i32(lens), 0.1, kv_idx=kv))


# More sequences than a wavefront's lanes and a workgroup's threads, most of them without a key, in
# tables from one page to many; lists of as many rows.
@pytest.mark.parametrize("B,width", [(65, 40), (300, 70), (300, 2), (700, 20)])
def test_decode_many_sequences(hip_lib, B, width):
    g = gen(B)
    lens = [0] * B
    for i in list(range(0, B, 97)) + [B - 1, B // 2, B // 2 + 1]:
        lens[i] = min(64 * width, 1 + (i * 37) % 2500)
    lens[B // 3] = 64 * width
    table, P = tables(lens, g, width=width)
    cache = filled(g, P, 2, 64, BF, B % 2 == 0)
    q = torch.randn(B, 6, 1, 64, generator=g, device=DEV).to(BF)
    out = check_decode(q, cache, table, lens, 0.125)
    assert (out[torch.tensor(lens, device=DEV) == 0] == 0).all()
    nb = torch.tensor([(n + 63) // 64 for n in lens], device=DEV)
    kv = torch.arange(width, device=DEV, dtype=torch.int32).view(1, 1, -1).repeat(B, 2, 1)
    counts = torch.stack([nb, (nb + 1) // 2], 1).to(torch.int32)
    check_decode(q, cache, table, lens, 0.125, kv_idx=kv, counts=counts)
    assert torch.equal(pc.paged_decode(q, cache, table, i32(lens), 0.125, kv_idx=kv)[:, :, :3],
                       pc.paged_decode(q, cache, table, i32(lens), 0.125, kv_idx=kv, counts=counts)[:, :, :3])


@pytest.mark.parametrize("e4m3", [False, True])
def test_decode_absent_pages_and_lengths(hip_lib, e4m3):
    cache = filled(gen(8), 6, 2, 128, BF, e4m3)
    q = torch.randn(4, 8, 1, 128, generator=gen(9), device=DEV).to(BF)
    table = i32([[0, -1, 6, 2, 3], [-1, -1, -1, -1, -1], [4, 5, 1, 0, 2], [1, 2, 3, 4, 5]])
    out = check_decode(q, cache, table, [300, 300, 1 << 30, -3], 0.1)
    assert (out[1] == 0).all() and (out[3] == 0).all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_decode_special_values(hip_lib, e4m3):
    """NaN keys touch their own KV head only; keys of score -inf weigh nothing; a row of nothing
    else gives zeros; an infinite value stays infinite."""
    g = gen(10)
    cache = filled(g, 6, 2, 128, FH, e4m3)
    table, lens = i32([[3, 1, 5]]), [170]
    q = torch.randn(1, 8, 1, 128, generator=g, device=DEV).to(FH)
    keep = check_decode(q, cache, table, lens, 0.1).clone()
    cache.k_pages[1, 1, 7, 3] = NAN
    out = pc.paged_decode(q, cache, table, i32(lens), 0.1)
    assert torch.equal(out[:, :, :4], keep[:, :, :4]) and out[:, :, 4:].isnan().all()
    if e4m3:
        return                                            # no infinities there
    cache = filled(g, 6, 2, 128, FH, False)
    q[..., 0] = 1.0
    cache.k_pages[3, :, :, 0] = -INF                       # the whole first page
    ref, mass = decode_ref(q, cache, i32([[1, 5]]), [170 - 64], 0.1)
    out = pc.paged_decode(q, cache, table, i32(lens), 0.1)
    check_close(out, ref, mass, FH)
    assert (pc.paged_decode(q, cache, table, i32([64]), 0.1) == 0).all()
    cache.v_pages[1, 0, 2, 5] = INF
    out = pc.paged_decode(q, cache, table, i32(lens), 0.1)
    assert torch.isposinf(out[0, 0, :4, 5]).all() and torch.isfinite(out[0, 0, 4:]).all()


def test_decode_shared_pages_and_sharp_scores(hip_lib):
    """Two sequences over one prefix; scores far apart, whose maximum comes late or early."""
    g = gen(11)
    cache = filled(g, 20, 2, 128, BF, True)
    table = i32([list(range(10)), list(range(8)) + [15, 16]])
    q = torch.randn(2, 8, 1, 128, generator=g, device=DEV).to(BF)
    check_decode(q, cache, table, [640, 600], 0.09)
    for where in (0, 639, 300):
        cache.k_scale.fill_(119)
        cache.k_scale[where // 64, :, where % 64] = 124
        check_decode(q, cache, table, [640, 640], 0.09)


def test_pages_past_32_bit_offsets(hip_lib):
    """A pool of more than 2^32 bytes of K: pages at its end."""
    P, Hk, D = 33000, 8, 128
    for e4m3, P in ((True, 66000), (False, 33000)):
        cache = pc.PagedCache.empty(P, Hk, D, BF, DEV, e4m3=e4m3)
        assert cache.k_pages.numel() > 1 << 31 and cache.k_pages.nbytes > 1 << 32
        g = gen(12)
        k, v = (torch.randn(150, Hk, D, generator=g, device=DEV).to(BF) for _ in range(2))
        table = i32([[P - 1, P - 2, P - 3]])
        pc.paged_write(cache, k, v, table, i32([0]), cu_new=i32([0, 150]))
        rk, rv = pc.paged_read(cache, table, i32([150]), 150)
        small = pc.PagedCache.empty(3, Hk, D, BF, DEV, e4m3=e4m3)
        near = i32([[2, 1, 0]])
        pc.paged_write(small, k, v, near, i32([0]), cu_new=i32([0, 150]))
        sk, sv = pc.paged_read(small, near, i32([150]), 150)
        assert torch.equal(rk, sk) and torch.equal(rv, sv)
        q = torch.randn(1, 16, 1, D, generator=g, device=DEV).to(BF)
        assert torch.equal(pc.paged_decode(q, cache, table, i32([150]), 0.1),
                           pc.paged_decode(q, small, near, i32([150]), 0.1))
        a, b = (pc.paged_select(q, c, t, i32([150]), 0.1, 3, 3) for c, t in ((cache, table), (small, near)))
        assert torch.equal(a.kv_idx, b.kv_idx)
        assert torch.equal(cache.planes[P - 3:], small.planes)
        del cache


# ---- together -----------------------------------------------------------------------------------

def test_generation_over_the_cache(hip_lib):
    """A prompt written, then tokens generated one by one: full decode equals the contiguous cache's
    to rounding, the listed one the definition over the selected pages, all read back at the end."""
    g = gen(13)
    H, Hk, D, scale = 8, 2, 128, 128 ** -0.5
    lens = [700, 65, 0, 1279]
    B, steps = len(lens), 70
    final = [n + steps for n in lens]
    table, P = tables(final, g)
    kall, vall = (torch.randn(B, Hk, max(final), D, generator=g, device=DEV).to(BF) for _ in range(2))
    for e4m3 in (False, True):
        cache = pc.PagedCache.empty(P, Hk, D, BF, DEV, e4m3=e4m3)
        packed = [torch.cat([x[b, :, :n].transpose(0, 1) for b, n in enumerate(lens)]) for x in (kall, vall)]
        seq = i32(lens)
        pc.paged_write(cache, *packed, table, i32([0] * B), cu_new=i32([sum(lens[:i]) for i in range(B + 1)]))
        for step in range(steps):
            k1, v1 = (torch.stack([x[b, :, n + step] for b, n in enumerate(lens)]) for x in (kall, vall))
            pc.paged_write(cache, k1, v1, table, seq)
            seq += 1
            if step % 23 and step != steps - 1:
                continue
            now = [n + step + 1 for n in lens]
            q = torch.randn(B, H, 1, D, generator=g, device=DEV).to(BF)
            sel = check_select(q, cache, table, now, scale, 4, 8, 0.2)
            check_decode(q, cache, table, now, scale, kv_idx=sel.kv_idx, counts=sel.counts)
            out = check_decode(q, cache, table, now, scale)
            for b, n in enumerate(now):
                dense = decode_attn(q[b:b + 1], kall[b:b + 1, :, :n], vall[b:b + 1, :, :n], scale)
                if not e4m3:
                    ref, mass = decode_ref(q[b:b + 1], cache, table[b:b + 1], [n], scale)
                    check_close(out[b:b + 1], dense.double(), mass, BF, times=2)
        k, v = pc.paged_read(cache, table, seq, max(final))
        for b, n in enumerate(final):
            for got, x in ((k, kall), (v, vall)):
                want = x[b, :, :n].double()
                if e4m3:
                    val, byte = e4m3_ref(want, BF)
                    want = val * torch.exp2(byte.double() - 127).unsqueeze(-1)
                assert torch.equal(got[b, :, :n].double(), want)
                assert (got[b, :, n:] == 0).all()


@pytest.mark.parametrize("e4m3", [False, True])
def test_decode_step_in_a_graph(hip_lib, e4m3):
    """A captured step (write, select, decode, read) replayed as the sequences grow, with eager work
    and synchronizations between, equals the eager step each time; on a stream of its own."""
    g = gen(14)
    H, Hk, D, scale = 16, 2, 128, 0.09
    lens = [900, 62, 1]
    table, P = tables([n + 8 for n in lens], g, width=64)
    caches = [filled(gen(15), P, Hk, D, BF, e4m3) for _ in range(2)]
    k, v = (torch.empty(3, Hk, D, dtype=BF, device=DEV) for _ in range(2))
    q, seq = torch.empty(3, H, 1, D, dtype=BF, device=DEV), i32(lens)

    def step(cache, seq):
        pc.paged_write(cache, k, v, table, seq)
        after = seq + 1
        s = pc.paged_select(q, cache, table, after, scale, 4, 9, tau=0.2)
        return (s.kv_idx, s.counts, s.sigma, s.uncertain, pc.paged_decode(q, cache, table, after, scale),
                pc.paged_decode(q, cache, table, after, scale, s.kv_idx, s.counts),
                *pc.paged_read(cache, table, after, 1000))

    def fresh(i):
        gi = gen(100 + i)
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gi, device=DEV))

    fresh(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0], seq)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(caches[0], seq)
    for i in range(5):
        fresh(i)
        want = step(caches[1], seq)
        torch.cuda.synchronize()
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        for name in ("k_pages", "v_pages", "k_scale", "v_scale", "planes"):
            a, b = (getattr(c, name) for c in caches)
            assert a is None or torch.equal(bits(a), bits(b)), (i, name)
        seq += 1


def test_two_streams_at_once(hip_lib):
    """Calls on two streams share nothing but what they read."""
    g = gen(16)
    table, P = tables([3000, 2000], g)
    cache = filled(g, P, 2, 128, BF, False)
    seq, scale = i32([3000, 2000]), 0.09
    qs = [torch.randn(2, 8, 1, 128, generator=g, device=DEV).to(BF) for _ in range(2)]
    want = [(pc.paged_decode(q, cache, table, seq, scale),
             pc.paged_select(q, cache, table, seq, scale, 5, 9, tau=0.1).kv_idx) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append((pc.paged_decode(qs[i], cache, table, seq, scale),
                               pc.paged_select(qs[i], cache, table, seq, scale, 5, 9, tau=0.1).kv_idx))
    torch.cuda.synchronize()
    for i in range(2):
        for out, idx in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(idx, want[i][1])


def test_refusals(hip_lib):
    cache = filled(gen(17), 4, 2, 128, BF, True)
    table, seq = i32([[0, 1]]), i32([100])
    q = torch.randn(1, 4, 1, 128, device=DEV).to(BF)
    k = torch.randn(1, 2, 128, device=DEV).to(BF)
    bad = [lambda: pc.paged_decode(q.half(), cache, table, seq, 0.1),
           lambda: pc.paged_decode(q[:, :3], cache, table, seq, 0.1),
           lambda: pc.paged_decode(q[..., :64], cache, table, seq, 0.1),
           lambda: pc.paged_decode(q, cache, table.long(), seq, 0.1),
           lambda: pc.paged_decode(q, cache, table, seq.long(), 0.1),
           lambda: pc.paged_decode(q, cache, table, seq.cpu(), 0.1),
           lambda: pc.paged_decode(q, cache, table, i32([1, 2]), 0.1),
           lambda: pc.paged_decode(q, cache, table, seq, float("nan")),
           lambda: pc.paged_decode(q, cache, table, seq, 0.1, counts=i32([[1, 1]])),
           lambda: pc.paged_decode(q, cache, table, seq, 0.1, kv_idx=i32([[[0]]])),
           lambda: pc.paged_decode(q, cache, table, seq, 0.1, out=torch.empty(1, 1, 4, 128, device=DEV)),
           lambda: pc.paged_decode(q.clone().requires_grad_(), cache, table, seq, 0.1),
           lambda: pc.paged_select(q, cache, table, seq, 0.1, 2, 4),
           lambda: pc.paged_select(q, cache, table, seq, 0.1, 5, 4),
           lambda: pc.paged_select(q, cache, table, seq, -0.1, 3, 4),
           lambda: pc.paged_select(q, cache, table, seq, 0.1, 3, 4, tau=float("nan")),
           lambda: pc.paged_write(cache, k.half(), k, table, seq),
           lambda: pc.paged_write(cache, k, k[:, :1], table, seq),
           lambda: pc.paged_write(cache, k[:0], k[:0], table, seq),
           lambda: pc.paged_write(cache, k, k, table, seq, cu_new=i32([0])),
           lambda: pc.paged_read(cache, table, seq, 0),
           lambda: pc.paged_read(cache, table, seq, 5, out=(k, k)),
           lambda: pc.PagedCache(cache.k_pages, cache.v_pages, dtype=BF),
           lambda: pc.PagedCache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale),
           lambda: pc.PagedCache(cache.k_pages[..., :96], cache.v_pages[..., :96], cache.k_scale, cache.v_scale, dtype=BF),
           lambda: pc.PagedCache(cache.k_pages, cache.v_pages, cache.k_scale, cache.v_scale, cache.planes, FH),
           lambda: pc.PagedCache(None, None)]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            print("not refused:", i)
    # read as their values: strided and negated views
    for x in (q.transpose(2, 3).contiguous().transpose(2, 3), torch._neg_view(-q)):
        assert torch.equal(pc.paged_decode(x, cache, table, seq, 0.1), pc.paged_decode(q, cache, table, seq, 0.1))


# ---- selection at the ends of the score range ---------------------------------------------------

def cut_ref(score, scale, k_base, k_slots, tau, NB):
    """(list, count, sigma, flag) of one row from its pages' fp64 scores; NaN ranks first."""
    nb = len(score)
    order = sorted(range(1, nb - 1), key=lambda j: (0, 0, j) if math.isnan(score[j]) else (1, -score[j], j))
    keep, k, sigma = min(k_base, nb), k_base - 2, 2.0
    if nb > k_base:
        first, last, below = (score[order[i]] * scale for i in (0, k - 1, k))
        gap, reach = last - below, first - below
        sigma = NAN if math.isnan(gap) or math.isnan(reach) or math.isinf(gap) else \
            min(max(gap / max(reach, 1e-9), 0.0), 2.0)
        if sigma < tau:
            keep = min(k_slots, nb)
    kept = list(range(nb)) if nb <= keep else sorted([0, nb - 1] + order[:keep - 2])
    return kept + [NB] * (k_slots - len(kept)), keep, sigma, int(sigma < tau)


def page_scores(q, planes, table):
    """fp64 scores [Hk, pages] of one sequence by the definition; absent pages are -inf."""
    Hk, P = planes.shape[1], planes.shape[0]
    there = (table >= 0) & (table < P)
    pl = planes[table.clamp(0, P - 1).long()].double().transpose(0, 1)            # [Hk, pages, 2, D]
    x = q.view(Hk, -1, q.shape[-1]).double()                                      # [Hk, G, D]
    s = torch.stack([torch.where(x[:, i:i + 1] >= 0, x[:, i:i + 1] * pl[:, :, 0],
                                 x[:, i:i + 1] * pl[:, :, 1]).sum(-1) for i in range(x.shape[1])]).amax(0)
    return torch.where(there, s, -INF)


def select_guarded(q, cache, table, lens, scale, k_base, k_slots, tau):
    """(kv_idx, counts, sigma, uncertain) through the C ABI, the lists between guard values."""
    B, H, _, D = q.shape
    Hk, NB, lib = cache.planes.shape[1], table.shape[1], _capi.lib()
    n = B * Hk * k_slots
    wide = torch.full((n + 8192,), -77, dtype=torch.int32, device=DEV)
    lists = wide[4096:4096 + n]
    counts = torch.empty(B, Hk, dtype=torch.int32, device=DEV)
    sigma = torch.empty(B, Hk, device=DEV)
    flags = torch.empty(B, Hk, dtype=torch.uint8, device=DEV)
    ws = torch.empty(lib.ugbsa_paged_select_workspace_elems(B, Hk, NB), device=DEV)
    _capi.check(lib.ugbsa_paged_select(
        cache._call[0], q.data_ptr(), *q.stride(), H, lens.data_ptr(), table.data_ptr(), table.stride(0), B,
        NB, scale, k_base, k_slots, tau, lists.data_ptr(), counts.data_ptr(), sigma.data_ptr(),
        flags.data_ptr(), ws.data_ptr(), ws.numel(), _capi.stream_ptr(DEV)), "paged_select")
    assert (wide[:4096] == -77).all() and (wide[4096 + n:] == -77).all()
    return lists.view(B, Hk, k_slots), counts, sigma, flags


def check_cut(q, cache, table, lens, scale, k_base, k_slots, tau):
    got = select_guarded(q, cache, table, i32(lens), scale, k_base, k_slots, tau)
    for b, n in enumerate(lens):
        nb = (n + 63) // 64
        score = page_scores(q[b, :, 0], cache.planes, table[b, :nb]).tolist()
        for h, row in enumerate(score):
            kept, keep, sigma, flag = cut_ref(row, scale, k_base, k_slots, tau, table.shape[1])
            assert got[0][b, h].tolist() == kept, (b, h)
            assert (int(got[1][b, h]), int(got[3][b, h])) == (keep, flag), (b, h)
            s = float(got[2][b, h])
            assert math.isnan(s) == math.isnan(sigma) and not abs(s - sigma) > 2.0 ** -24 * sigma + 1e-12, (b, h)


# Rows of every form of the pick (128, 256 and 512 threads with their keys in registers, and longer).
@pytest.mark.parametrize("nb", [60, 1500, 3000, 5000])
@pytest.mark.parametrize("value", [INF, NAN])
def test_select_cut_among_infinite_and_nan_pages(hip_lib, nb, value):
    """Fewer, as many and more such pages than the list has places, with and without absent pages."""
    print(f"[case] select among {value} pages nb={nb}", flush=True)
    g = gen(nb)
    k_base, k_slots = 8, 20
    for n in (1, 5, 6, 7, 18, 19, 40):
        for absent in (0, 3):
            cache = filled(g, 2 * nb + 1, 2, 64, BF, False)
            table = torch.randperm(2 * nb, generator=g, device=DEV).view(2, nb).int()
            q = torch.randn(2, 6, 1, 64, generator=g, device=DEV).to(BF)
            q[..., 0] = 1.0
            for h in range(2):
                at = table[:, 1:nb - 1].gather(1, torch.rand(2, nb - 2, generator=g, device=DEV).argsort(1)[:, :n])
                cache.planes[at[0].long(), h, 0, 0] = value
                cache.planes[at[1, :n - h].long(), h, 0, 0] = value
            table[:, 2:2 + absent] = -1
            check_cut(q, cache, table, [64 * nb, 64 * nb - 63], 0.125, k_base, k_slots, 0.05)


def test_select_sigma_of_one_nan_page(hip_lib):
    """The page ranks first and the cut lies among finite scores: sigma is NaN, below no tau."""
    g = gen(23)
    cache = filled(g, 40, 1, 64, BF, False)
    cache.planes[17, 0, :, 5] = NAN
    q = torch.randn(1, 4, 1, 64, generator=g, device=DEV).to(BF)
    r = pc.paged_select(q, cache, torch.arange(40, device=DEV, dtype=torch.int32).view(1, 40), i32([40 * 64]),
                        0.125, 8, 16, tau=3.0)
    assert r.sigma.isnan().all() and r.uncertain.tolist() == [[0]] and r.counts.tolist() == [[8]]
    assert 17 in r.kv_idx[0, 0].tolist()


def test_select_of_a_nan_query(hip_lib):
    """Every page's score is NaN but an absent one's; the other sequence's list is its own."""
    g = gen(20)
    for nb in (70, 1100):
        cache = filled(g, 2 * nb, 1, 64, FH, False)
        table = torch.arange(2 * nb, device=DEV, dtype=torch.int32).view(2, nb)
        table[0, 9] = -1
        q = torch.randn(2, 4, 1, 64, generator=g, device=DEV).to(FH)
        q[0, :, :, 3] = NAN
        check_cut(q, cache, table, [64 * nb, 64 * nb], 0.125, 64, 66, 0.05)


# A cut whose first bin holds more keys than a workgroup has threads is looked for in it again.
@pytest.mark.parametrize("nb", [600, 1500, 3000, 5000])
def test_select_cut_among_near_equal_scores(hip_lib, nb):
    cache = filled(gen(21), nb, 1, 64, BF, False)
    i = torch.randperm(nb, generator=gen(22), device=DEV)
    cache.planes[:] = 0.0
    cache.planes[:, :, :, 0] = 1.0
    cache.planes[:, 0, :, 1] = ((i % 256) * 2.0 ** -30).to(BF).unsqueeze(-1)      # all exact in fp64
    cache.planes[:, 0, :, 2] = ((i // 256) * 2.0 ** -22).to(BF).unsqueeze(-1)
    q = torch.ones(1, 2, 1, 64, device=DEV, dtype=BF)
    for far in (2.0 ** 100, -2.0 ** 100):
        cache.planes[nb // 2, :, :, 3] = far
        table = torch.arange(nb, device=DEV, dtype=torch.int32).view(1, nb)
        for k_base, k_slots, tau in ((5, 9, 0.0), (400, 500, 1.5), (580, 590, 0.0)):
            check_cut(q, cache, table, [64 * nb], 0.125, k_base, k_slots, tau)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads", [1, 5, 9])
def test_select_bounds_of_different_magnitude(hip_lib, D, heads):
    """The bound that a dim does not take is 2^60 times the one it takes: no part of the score.  The
    scores are whole numbers, so their sums are exact in any order."""
    g = gen(D + heads)
    nb = 40
    cache = filled(g, nb, 2, D, BF, False)
    small = torch.randint(-8, 9, (nb, D), generator=g, device=DEV).to(BF)
    huge = (2.0 ** 60 * torch.randint(1, 9, (nb, D), generator=g, device=DEV)).to(BF)
    cache.planes[:, 0, 0], cache.planes[:, 0, 1] = small, -huge        # taken by q >= 0
    cache.planes[:, 1, 0], cache.planes[:, 1, 1] = huge, small         # taken by q < 0
    q = torch.randint(1, 9, (1, 2 * heads, 1, D), generator=g, device=DEV).to(BF)
    q[:, heads:] *= -1
    table = torch.arange(nb, device=DEV, dtype=torch.int32).view(1, nb)
    for k_base, k_slots, tau in ((6, 12, 0.02), (20, 30, 0.0)):
        check_cut(q, cache, table, [64 * nb], 0.125, k_base, k_slots, tau)


def test_pages_that_share_memory_are_read_only(hip_lib):
    """Expanded pages, or one tensor for K and V: attended to and read back, not written."""
    g = gen(24)
    full = filled(g, 3, 2, 64, BF, False)
    table, seq = i32([[2, 0]]), i32([100])
    q, k1 = torch.randn(1, 4, 1, 64, generator=g, device=DEV).to(BF), torch.zeros(1, 2, 64, device=DEV, dtype=BF)
    for k, v in ((full.k_pages[:, :1].expand(3, 2, 64, 64), full.v_pages), (full.k_pages, full.k_pages)):
        shared, own = pc.PagedCache(k, v), pc.PagedCache(k.contiguous(), v.clone())
        assert torch.equal(pc.paged_decode(q, shared, table, seq, 0.1), pc.paged_decode(q, own, table, seq, 0.1))
        for a, b in zip(pc.paged_read(shared, table, seq, 100), pc.paged_read(own, table, seq, 100)):
            assert torch.equal(a, b)
        with pytest.raises(AssertionError, match="share memory"):
            pc.paged_write(shared, k1, k1, table, seq)
        pc.paged_write(own, k1, k1, table, seq)


# ---- branches that take large calls ---------------------------------------------------------------

# The pages that a table's width admits are more than 768 MB: they are read past the cache.
@pytest.mark.parametrize("H,Hk,D,dtype,e4m3", [(6, 2, 64, BF, False), (6, 2, 64, FH, True), (28, 4, 128, BF, False),
                                               (8, 2, 128, FH, True), (8, 2, 128, FH, False), (16, 2, 256, BF, True),
                                               (8, 2, 128, BF, True), (16, 2, 256, FH, False), (6, 2, 64, FH, False),
                                               (6, 2, 64, BF, True), (16, 2, 256, BF, False), (16, 2, 256, FH, True)])
def test_decode_of_tables_wide_enough_to_stream(hip_lib, H, Hk, D, dtype, e4m3):
    print(f"[case] streamed decode H={H}/{Hk} D={D} {dtype} {e4m3}", flush=True)
    g = gen(D + H)
    lens = [1500, 0, 700]
    width = (768 << 20) // (len(lens) * Hk * 2 * 64 * D * (1 if e4m3 else 2)) + 1
    table, P = tables(lens, g, width=width)
    cache = filled(g, P, Hk, D, dtype, e4m3)
    q = torch.randn(len(lens), H, 1, D, generator=g, device=DEV).to(dtype)
    check_decode(q, cache, table, lens, D ** -0.5)


# An output of 256 MiB or more is written past the cache, and its pages read past it.
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("e4m3", [False, True])
def test_read_of_lengths_long_enough_to_stream(hip_lib, D, dtype, e4m3):
    g = gen(D)
    lens, Hk = [1000, 64, 0, 333], 4
    table, P = tables(lens, g)
    cache = filled(g, P, Hk, D, dtype, e4m3)
    n = (256 << 20) // (4 * len(lens) * Hk * D) + 3
    near = pc.paged_read(cache, table, i32(lens), 1000)
    for a, b in zip(pc.paged_read(cache, table, i32(lens), n), near):
        assert torch.equal(a[:, :, :1000], b) and not a[:, :, 1000:].any()


@pytest.mark.parametrize("nb", [1024, 1025, 1500, 2048, 2049, 3000, 4096, 4097])
def test_select_at_the_sizes_of_the_pick(hip_lib, nb):
    """Rows of 128, 256 and 512 threads with keys in registers, and of more."""
    g = gen(nb)
    cache = filled(g, nb, 2, 64, BF, False)
    table = torch.stack([torch.randperm(nb, generator=g, device=DEV) for _ in range(2)]).int()
    q = torch.randn(2, 8, 1, 64, generator=g, device=DEV).to(BF)
    for k_base, k_slots, tau in ((64, 128, 0.005), (256, 300, 0.0), (3, 9, 9.0), (nb - 1, nb, 1e-4)):
        check_cut(q, cache, table, [64 * nb - 7, 64 * (nb // 2)], 0.125, k_base, k_slots, tau)


# ---- lengths that go back -------------------------------------------------------------------------

@pytest.mark.parametrize("e4m3", [False, True])
def test_planes_after_a_shorter_length(hip_lib, e4m3):
    """Tokens taken back and others written in their place: the planes bound the keys that were given
    for every token that is left, and a page that starts again at slot 0 forgets the old ones."""
    g = gen(25)
    cache = filled(g, 5, 2, 128, BF, e4m3)
    table = i32([[3, 0, 4]])
    keys = 4 * torch.randn(190, 2, 128, generator=g, device=DEV).to(BF)
    pc.paged_write(cache, keys, keys, table, i32([0]), cu_new=i32([0, 190]))
    for back, n in ((100, 20), (64, 1), (63, 90)):
        new = torch.randn(n, 2, 128, generator=g, device=DEV).to(BF)
        keys = torch.cat([keys[:back], new])
        pc.paged_write(cache, new, new, table, i32([back]), cu_new=i32([0, n]))
        for j in range((len(keys) + 63) // 64):
            page, held = int(table[0, j]), keys[64 * j:64 * j + 64]
            assert (cache.planes[page, :, 0] >= held.amax(0)).all() and (cache.planes[page, :, 1] <= held.amin(0)).all()
            if 64 * j >= back:
                assert torch.equal(cache.planes[page, :, 0], held.amax(0))
                assert torch.equal(cache.planes[page, :, 1], held.amin(0))


def test_contiguous_decode_over_what_is_read_back(hip_lib):
    """The cache read back is the dispatcher's layout: its decode attends to it as the paged one does."""
    g = gen(26)
    table, P = tables([777], g)
    for e4m3 in (False, True):
        cache = filled(g, P, 2, 128, BF, e4m3)
        q = torch.randn(1, 8, 1, 128, generator=g, device=DEV).to(BF)
        k, v = pc.paged_read(cache, table, i32([777]), 777)
        ref, mass = decode_ref(q, cache, table, [777], 0.09)
        out, _ = sa.block_sparse_attention(None, q, k, v, None, 0.09)
        check_close(out, ref, mass, BF)
        check_close(pc.paged_decode(q, cache, table, i32([777]), 0.09), ref, mass, BF)


def test_calls_repeat_themselves(hip_lib):
    """The same call gives the same bits: no result depends on the order in which workgroups end."""
    g = gen(27)
    lens = [3000, 1, 0, 9000, 640, 70] * 9
    table, P = tables(lens, g)
    for dtype, e4m3 in ((BF, False), (FH, True)):
        cache = filled(g, P, 2, 128, dtype, e4m3)
        q = torch.randn(len(lens), 8, 1, 128, generator=g, device=DEV).to(dtype)
        first = pc.paged_decode(q, cache, table, i32(lens), 0.09)
        sel = pc.paged_select(q, cache, table, i32(lens), 0.09, 8, 16, tau=0.1)
        part = pc.paged_decode(q, cache, table, i32(lens), 0.09, sel.kv_idx, sel.counts)
        for _ in range(5):
            assert torch.equal(first, pc.paged_decode(q, cache, table, i32(lens), 0.09))
            again = pc.paged_select(q, cache, table, i32(lens), 0.09, 8, 16, tau=0.1)
            assert torch.equal(sel.kv_idx, again.kv_idx) and torch.equal(sel.sigma, again.sigma)
            assert torch.equal(part, pc.paged_decode(q, cache, table, i32(lens), 0.09, sel.kv_idx, sel.counts))


@pytest.mark.parametrize("heads", [1, 4, 5, 7, 8])
def test_select_zeros_of_either_sign_take_the_upper_bound(hip_lib, heads):
    """q = -0 is >= 0: its bound is K-max, which shows where one of the bounds is infinite."""
    g = gen(heads)
    nb = 30
    cache = filled(g, nb, 2, 64, BF, False)
    q = torch.randn(1, 2 * heads, 1, 64, generator=g, device=DEV).to(BF)
    q[..., 7], q[..., 8] = -0.0, 0.0
    cache.planes[3, 0, 0, 7] = cache.planes[4, 0, 0, 8] = INF                 # NaN scores
    cache.planes[5, :, 1, 7] = cache.planes[6, :, 1, 8] = -INF                # not looked at
    table = torch.arange(nb, device=DEV, dtype=torch.int32).view(1, nb)
    check_cut(q, cache, table, [64 * nb], 0.125, 4, 8, 0.1)
    check_cut(q, cache, table, [64 * nb], 0.125, 9, 12, 0.1)
