"""What rotary positions, the 4-bit paged cache and eviction are measured on: inputs, plain forms, costs.

Around the paged key-value cache (pages of 64 tokens that a block table names), serving needs

* ``rotary``: queries and keys turned by their positions, pairs of dims by angle pos * f_j: half or
  interleaved pairs, all of a head or its first dims, frequencies plain or scaled for long contexts;
  with its gradient;
* ``write``: new tokens into the cache, the keys turned on the way where the case says so, or
  quantised to e2m1 (two codes a byte, a power-of-two scale per 32 dims of a token's head:
  ``k_pages`` / ``v_pages`` [P, Hk, 64, D / 2], ``k_scale`` / ``v_scale`` [P, Hk, D / 32, 64] uint8, the
  value being code * 2^(scale - 127)); quantised tokens are read back as values;
* ``decode``: attention of one new token over an e2m1 cache;
* ``mass``: the same over any cache, the weights that each cached token gets added up over the query
  heads of its KV head;
* ``evict``: per sequence and KV head the first, the newest and the heaviest tokens kept, packed into
  other pages with their scales, weights and page summaries.

Where ``own`` is true a pass makes the package's calls; otherwise it computes the operator from
elementary torch operations in 32 bits (64 for angles).
"""

import math
import os
import random
import sys

import torch

own = False

PAGE = 64
GROUP = 32                 # dims that share an e2m1 scale
DEV = "cuda"
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                   "uncertainty-gated-block-sparse-attention_amd")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# The largest magnitude that reads back finite from two significant bits
LARGEST = {"bf16": 1.5 * 2.0 ** 127, "fp16": 49152.0}


def _case(op, name=None, **kw):
    base = dict(op=op, B=1, H=28, Hk=4, D=128, dtype="bf16")
    if op == "rotary" or kw.get("turned"):
        # rotary dims, layout, frequencies; the first position of the longest sequence
        base.update(rot=128, interleaved=False, scaling="none", start=1000)
    if op == "rotary":
        base.update(M=1, grad=False)                  # tokens of a sequence
    else:
        base.update(cache="e2m1", length=1000, ragged=False)
    if op == "write":
        base.update(new=1, turned=False)              # new tokens of the longest sequence
    if op == "evict":
        base.update(keep=512, recent=64, first=4)
    base.update(kw)
    return {"name": name, **base} if name else base


def listed():
    return [
        # query and key of one generated token: launch latency
        _case("rotary", "rotary_one_token"),
        # a training step's layer: two long sequences of an odd length, scaled frequencies, gradients
        _case("rotary", "rotary_grad_b2_8k", B=2, H=40, Hk=8, M=8191, scaling="yarn", start=60000, grad=True),
        # a decode step of 192 sequences, interleaved pairs on part of the head, 16-bit cache
        _case("write", "write_turned_step_b192", B=192, H=40, Hk=8, cache="model", length=512, ragged=True,
              turned=True, rot=64, interleaved=True, scaling="linear", start=511),
        # two short prompts behind cached prefixes, head_dim 64, fp16, into four bits and back
        _case("write", "write_chunk_hd64_fp16", B=2, H=16, D=64, dtype="fp16", length=1999, new=77, ragged=True),
        # six prompts of up to 16K tokens into four bits and back
        _case("write", "write_prompts_e2m1", B=6, length=777, new=16384, ragged=True),
        # one short sequence: the latency of a decode step's attention
        _case("decode", "decode_1k"),
        # a mixed batch of up to 16K tokens a sequence, head_dim 256, fp16
        _case("decode", "decode_b24_16k_hd256_fp16", B=24, H=16, Hk=2, D=256, dtype="fp16", length=16384,
              ragged=True),
        # the largest: 32 sequences of 64K tokens
        _case("decode", "decode_b32_64k", B=32, H=40, Hk=8, length=65536),
        # one sequence of a 16-bit cache whose weights are followed
        _case("mass", "mass_4k", cache="model", length=4096),
        # an ordinary batch from four bits, up to 32K tokens
        _case("mass", "mass_b16_32k", B=16, H=40, Hk=8, length=32768, ragged=True),
        # one short sequence cut back to its budget
        _case("evict", "evict_600", cache="model", length=600),
        # eight sequences of up to 32K tokens, quantised, an eighth of the longest kept
        _case("evict", "evict_b8_32k_e4m3", B=8, H=40, Hk=8, cache="e4m3", length=32768, ragged=True, keep=4000,
              recent=500),
    ]


_SHAPES = [(28, 4, 128), (40, 8, 128), (8, 2, 128), (16, 2, 256), (16, 4, 64), (8, 8, 64), (34, 2, 128)]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _turns(rng, D):
    return dict(rot=rng.choice([D, D, D // 2, 2 * rng.randrange(1, D // 2)]), interleaved=rng.random() < 0.5,
                scaling=rng.choice(["none", "linear", "ntk", "yarn"]), start=_log_int(rng, 1, 1 << 20))


def draw(rng):
    op = rng.choice(["rotary", "write", "decode", "decode", "mass", "evict"])
    H, Hk, D = rng.choice(_SHAPES)
    kw = dict(H=H, Hk=Hk, D=D, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "rotary":
        kw.update(B=_log_int(rng, 1, 64), M=rng.choice([1, _log_int(rng, 2, 32768)]), grad=rng.random() < 0.4,
                  **_turns(rng, D))
        if kw["rot"] < 4:
            kw["scaling"] = "none"
    else:
        kw.update(B=_log_int(rng, 1, 192), length=_log_int(rng, 1, 131072), ragged=rng.random() < 0.7)
    if op == "write":
        kw.update(length=_log_int(rng, 1, 2048), new=rng.choice([1, _log_int(rng, 2, 16384)]))
        if rng.random() < 0.4:
            # not into fewer bits: a rotation that 32 bits round to either side of a border of 16 bits
            # may then lie to either side of one of 4 bits
            kw.update(turned=True, cache="model", **_turns(rng, D))
            if kw["rot"] < 4:
                kw["scaling"] = "none"
    if op == "mass":
        kw.update(cache=rng.choice(["model", "e4m3", "e2m1"]))
    if op == "evict":
        kw.update(cache=rng.choice(["model", "e4m3", "e2m1"]), length=_log_int(rng, 1, 65536))
        kw.update(keep=_log_int(rng, 1, 8192))
        kw.update(recent=rng.randrange(kw["keep"] // 4 + 1), first=rng.choice([0, min(4, kw["keep"] // 2)]))
    most = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    room = {"rotary": 1 << 29, "write": 1 << 28, "decode": 1 << 31, "mass": 1 << 29, "evict": 1 << 29}[op]
    c = _case(op, **kw)
    size = "new" if op == "write" else ("M" if op == "rotary" else "length")

    def over():
        # no more work, and no more to hold, than the largest listed call of the operator
        return work(c)["bytes"] > most or c["B"] * _longest(c) * (Hk if op != "rotary" else H) * D > room
    while c["B"] > 1 and over():
        c["B"] = c["B"] * 3 // 4
    while c[size] > 1 and over():
        c[size] = c[size] * 3 // 4
    return c


def _longest(c):
    return c["M"] if c["op"] == "rotary" else c["length"] + c.get("new", 0)


def _lengths(c):
    """(cached tokens, new tokens) of each sequence: a function of the case alone."""
    r = random.Random("%(B)d %(length)d %(ragged)s" % c)
    n = [c["length"]] * c["B"]
    new = [c.get("new", 0)] * c["B"]
    if c["ragged"]:
        # lengths over their logarithm, the longest as given; a slot without a sequence where the
        # batch has one to spare, and a first prompt with nothing cached
        n = [_log_int(r, max(1, c["length"] // 64), c["length"]) for _ in n]
        n[-1] = c["length"]
        if c["B"] > 4:
            n[1] = 0
        if c.get("new", 0) > 1:
            n[0] = 0
            new = [_log_int(r, max(1, c["new"] // 8), c["new"]) for _ in new]
            new[-1] = c["new"]
    return n, new


def _pages(n):
    return -(-n // PAGE)


def work(c):
    H, Hk, D = c["H"], c["Hk"], c["D"]
    if c["op"] == "rotary":
        one = c["B"] * c["M"] * (H + Hk) * D
        passes = 2 if c["grad"] else 1
        return {"bytes": passes * 4 * one + 4 * c["B"] * c["M"] + 8 * (c["rot"] // 2),
                "flops": passes * 3 * c["B"] * c["M"] * (H + Hk) * c["rot"]}
    n, new = _lengths(c)
    bits = {"model": 16 * D, "e4m3": 8 * D + 8, "e2m1": 4 * D + D // 4}[c["cache"]]
    token = 2 * Hk * bits // 8                                     # K and V of one cached token
    table = 4 * sum(_pages(a + b) for a, b in zip(n, new))
    if c["op"] == "write":
        touched = sum(_pages(a + b) - a // PAGE for a, b in zip(n, new))
        kept = sum(1 for a in n if a % PAGE)                       # summaries that are added to
        size = sum(new) * (4 * Hk * D + token) + (touched + kept) * 4 * Hk * D + table
        if c["cache"] == "e2m1":                                   # the cached tokens back
            size += sum(n) * token + c["B"] * _longest(c) * 4 * Hk * D
        return {"bytes": size, "flops": (9 if c["turned"] else 6) * sum(new) * Hk * D}
    if c["op"] == "evict":
        kept = [min(a, c["keep"]) for a in n]
        return {"bytes": sum(n) * 4 * Hk + sum(kept) * (2 * token + 8 * Hk) + sum(_pages(k) for k in kept) * 4 * Hk * D
                         + table, "flops": 2 * sum(n) * Hk}
    size = sum(n) * token + table + c["B"] * H * D * 4
    if c["op"] == "mass":
        size += sum(n) * 8 * Hk
    return {"bytes": size, "flops": 4 * sum(n) * H * D}


# ---- inputs ---------------------------------------------------------------------------------

def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


_SCALED = {"none": {}, "linear": dict(scaling="linear", factor=8.0), "ntk": dict(scaling="ntk", factor=8.0),
           "yarn": dict(scaling="yarn", factor=4.0, original=32768)}


def _cache_tensors(g, c, P, dt):
    """Pages as a cache holds them: normal keys and values, quantised where the cache is."""
    Hk, D, s = c["Hk"], c["D"], {}
    for name in ("k", "v"):
        if c["cache"] == "model":
            s[name + "_pages"] = _randn(g, P, Hk, PAGE, D, dtype=dt)
        elif c["cache"] == "e4m3":
            s[name + "_pages"] = (_randn(g, P, Hk, PAGE, D, dtype=torch.bfloat16) * 128).clamp_(
                -448, 448).to(torch.float8_e4m3fn)
            s[name + "_scale"] = torch.randint(118, 122, (P, Hk, PAGE), generator=g, device=DEV,
                                               dtype=torch.uint8)
        else:
            s[name + "_pages"] = torch.empty(P, Hk, PAGE, D // 2, dtype=torch.uint8, device=DEV)
            s[name + "_scale"] = torch.empty(P, Hk, D // GROUP, PAGE, dtype=torch.uint8, device=DEV)
            step = max(1, (1 << 27) // (Hk * PAGE * D))
            for p in range(0, P, step):
                x = _randn(g, min(step, P - p), Hk, PAGE, D, dtype=dt)
                code, e = _quantise(x, LARGEST[c["dtype"]])
                s[name + "_pages"][p : p + step] = code
                s[name + "_scale"][p : p + step] = e.transpose(2, 3)
    return s


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]
    B, H, Hk, D = c["B"], c["H"], c["Hk"], c["D"]
    s = dict(case=dict(c), dtype=dt, scale=D ** -0.5)
    if c["op"] == "rotary":
        M = c["M"]
        if c["grad"]:       # a layer's projections, heads side by side in each token
            s["q"], s["k"] = (_randn(g, B, M, h, D).to(dt).transpose(1, 2).requires_grad_() for h in (H, Hk))
            s["dq"], s["dk"] = (_randn(g, B, M, h, D).to(dt).transpose(1, 2) for h in (H, Hk))
            s["positions"] = c["start"] + torch.arange(M, device=DEV, dtype=torch.int32)
        else:               # packed tokens, q, k and v from one projection
            qkv = _randn(g, B * M, H + 2 * Hk, D).to(dt)
            s["q"], s["k"] = qkv[:, :H], qkv[:, H : H + Hk]
            begin = torch.randint(0, c["start"], (B, 1), generator=g, device=DEV)
            begin[-1] = c["start"]
            s["positions"] = (begin + torch.arange(M, device=DEV)).flatten().to(torch.int32)
        return s
    n, new = _lengths(c)
    held = [_pages(a + b) for a, b in zip(n, new)]
    after = [min(a, c["keep"]) for a in n] if c["op"] == "evict" else []
    fresh = [_pages(a) for a in after]
    width, P = max(max(held), 1), sum(held) + sum(fresh) + 3
    # pages in the order an allocator hands them out after some time: none in particular; entries
    # past a sequence's pages name no page
    free = torch.randperm(P, generator=g, device=DEV, dtype=torch.int32)

    def named(counts, first, wide):
        d = _i32(counts)
        at = first + (torch.cumsum(d, 0) - d).unsqueeze(1) + torch.arange(wide, device=DEV)
        return torch.where(torch.arange(wide, device=DEV) < d.unsqueeze(1), free[at.clamp(max=P - 1)],
                           -1).to(torch.int32)
    s.update(table=named(held, 0, width), lens=_i32(n), **_cache_tensors(g, c, P, dt))
    if c["op"] == "decode" or c["op"] == "mass":
        s["q"] = _randn(g, B, 1, H, D).to(dt).transpose(1, 2)      # [B, H, 1, D], as projected
    else:
        mid = _randn(g, P, Hk, D, dtype=dt)
        s["planes"] = torch.stack([mid + 1, mid - 1], 2).contiguous()
    if c["op"] == "write":
        T = sum(new)
        # projections of the packed new tokens, behind them the padding of the batch
        kv = _randn(g, T + 5, 2, Hk, D) * torch.exp(0.5 * _randn(g, T + 5, 2, Hk, 1))
        kv = kv.to(dt)
        s["k"], s["v"], s["total"] = kv[:, 0], kv[:, 1], T
        s["cu"] = _i32([sum(new[:i]) for i in range(B + 1)])
        s["after"] = _i32([a + b for a, b in zip(n, new)])
        if c["turned"]:     # positions behind tokens that were evicted before
            begin = [c["start"] + a for a in n]
            s["positions"] = _i32([p + i for p, m in zip(begin, new) for i in range(m)] + [0] * 5)
    if c["op"] in ("mass", "evict"):
        # weights gathered so far: most tokens next to none, a few most of it
        s["mass"] = torch.exp(2.5 * _randn(g, B, Hk, width * PAGE) - 6)
    if c["op"] == "evict":
        s["new_table"] = named(fresh, sum(held), max(_pages(c["keep"]), 1))
    return s


# ---- the package's calls --------------------------------------------------------------------

def _own(s):
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import paged_cache as pc
    import rotary as ro
    c = s["case"]
    turned = c["op"] == "rotary" or c.get("turned")
    if turned and "rot" not in s:      # the handle that a program keeps with its model
        s["rot"] = ro.Rotary.make(c["rot"], DEV, interleaved=c["interleaved"], **_SCALED[c["scaling"]])
    if c["op"] == "rotary":
        q, k = ro.rotary(s["rot"], s["positions"], s["q"], s["k"])
        if not c["grad"]:
            return q, k
        return (q, k) + torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    if "cache" not in s:               # the handle that a program keeps with its pages
        s["cache"] = pc.PagedCache(dtype=s["dtype"], **{k: s.get(k) for k in (
            "k_pages", "v_pages", "k_scale", "v_scale", "planes")})
    cache = s["cache"]
    if c["op"] == "write":
        turn = dict(rotary=s["rot"], positions=s["positions"]) if turned else {}
        pc.paged_write(cache, s["k"], s["v"], s["table"], s["lens"], cu_new=s["cu"], **turn)
        if c["cache"] != "e2m1":
            return _pools(s)
        return (s["planes"],) + pc.paged_read(cache, s["table"], s["after"], _longest(c))
    if c["op"] == "decode":
        return pc.paged_decode(s["q"], cache, s["table"], s["lens"], s["scale"])
    if c["op"] == "mass":
        mass = s["mass"].clone()       # a pass may be made again
        out = pc.paged_decode(s["q"], cache, s["table"], s["lens"], s["scale"], mass=mass)
        return {"out": out, "mass": mass}
    r = pc.paged_evict(cache, s["mass"], s["table"], s["lens"], s["new_table"], c["keep"], recent=c["recent"],
                       first=c["first"])
    pools = _pools(s) if c["cache"] != "e2m1" else dict(zip(("planes", "k", "v"), (s["planes"],) + pc.paged_read(
        cache, s["new_table"], r.seq_lens, c["keep"])))
    return {"kept": r.kept, "seq_lens": r.seq_lens, "mass": r.mass, **pools}


def _pools(s):
    return {k: s[k] for k in ("k_pages", "v_pages", "k_scale", "v_scale", "planes") if s.get(k) is not None}


# ---- plain forms ----------------------------------------------------------------------------

def _frequencies(c):
    """(f_j [rot / 2] fp64, what the turned values are multiplied by)."""
    r, how = c["rot"], dict(_SCALED[c["scaling"]])
    base, j = 10000.0, torch.arange(c["rot"] // 2, dtype=torch.float64, device=DEV)
    if c["scaling"] == "ntk":
        base = base * how["factor"] ** (r / (r - 2))
    f = base ** (-2 * j / r)
    if c["scaling"] == "linear":
        f = f / how["factor"]
    if c["scaling"] != "yarn":
        return f, 1.0
    # pairs that turn more than 32 times within the original context stay, those that turn less than
    # once are slowed down, the others lie between

    def pair(turns):
        return r * math.log(how["original"] / (2 * math.pi * turns)) / (2 * math.log(base))
    low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), r - 1)
    slow = ((j - low) / max(high - low, 0.001)).clamp(0, 1)
    return f * (1 - slow) + f / how["factor"] * slow, 0.1 * math.log(how["factor"]) + 1


def _turn(c, x, positions, back=False):
    """x [..., D] turned by positions (broadcast against x[..., 0]), in x's dtype."""
    f, m = _frequencies(c)
    angle = positions.double().unsqueeze(-1) * f
    cos, sin = (torch.cos(angle) * m).float(), (torch.sin(angle) * (-m if back else m)).float()
    r, y = c["rot"], x.float().clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    xa, xb = x[..., a].float(), x[..., b].float()
    y[..., a] = xa * cos - xb * sin
    y[..., b] = xb * cos + xa * sin
    return y.to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    if not c["grad"]:
        at = s["positions"].unsqueeze(1)
        return _turn(c, s["q"], at), _turn(c, s["k"], at)
    q, k = s["q"].detach(), s["k"].detach()
    return (_turn(c, q, s["positions"]), _turn(c, k, s["positions"]),
            _turn(c, s["dq"], s["positions"], back=True), _turn(c, s["dk"], s["positions"], back=True))


def _quantise(x, largest):
    """(packed codes [..., D / 2], scales [..., D / 32]) of x [..., D]: the smallest power of two that
    brings a group's largest finite magnitude to 6 or less, then the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6
    with halves to the even code; a group with a NaN has the scale 255."""
    x = x.float().unflatten(-1, (-1, GROUP)).clamp(-largest, largest)
    bits = torch.nan_to_num(x, nan=0.0).abs().amax(-1).view(torch.int32)
    e = (bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x400000).int()
    e = torch.where(bits == 0, 127, e.clamp(0, 254))
    y = torch.ldexp(x, (127 - e).unsqueeze(-1)).abs()
    # the code counts the steps below it: halves up to 2, ones up to 4, then 6
    code = torch.where(y < 2, torch.round(y * 2), torch.where(y < 4, torch.round(y) + 2, torch.round(y / 2) + 4))
    code = code.clamp(0, 7).nan_to_num(nan=0.0).to(torch.uint8) | (torch.signbit(x).to(torch.uint8) << 3)
    e = torch.where(x.isnan().any(-1), 255, e)
    code = code.flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), e.to(torch.uint8)


_CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _value(s, name, pages, heads):
    """[..., 64, D] fp32: the cached values of some pages of some heads."""
    x = s[name + "_pages"][pages, heads]
    if s["case"]["cache"] == "model":
        return x.float()
    e = (s[name + "_scale"][pages, heads].int() << 23).view(torch.float32)
    if s["case"]["cache"] == "e4m3":
        return x.float() * e.unsqueeze(-1)
    pairs = torch.tensor([[_CODES[i & 15], _CODES[i >> 4]] for i in range(256)], device=DEV)
    x = pairs[x.long()].flatten(-2)
    return (x.unflatten(-1, (-1, GROUP)) * e.transpose(-1, -2).unsqueeze(-1)).flatten(-2)


def _plain_write(s):
    c, T = s["case"], s["total"]
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(s["cu"], t.int(), right=True) - 1
    pos = s["lens"][b].long() + t - s["cu"][b]
    page, slot = s["table"][b, pos // PAGE].long(), pos % PAGE
    heads = torch.arange(c["Hk"], device=DEV)
    k = s["k"][:T]
    if c["turned"]:
        k = _turn(c, k, s["positions"][:T].unsqueeze(1))
    for name, x in (("k", k), ("v", s["v"][:T])):
        if c["cache"] == "e2m1":
            x, e = _quantise(x, LARGEST[c["dtype"]])
            group = torch.arange(c["D"] // GROUP, device=DEV)
            s[name + "_scale"][page[:, None, None], heads[:, None], group, slot[:, None, None]] = e
        s[name + "_pages"][page[:, None], heads, slot[:, None]] = x
    # a page that gets its first token starts over; the others add to what they have
    planes, x = s["planes"].float(), k.float()
    P = planes.shape[0]
    start = torch.zeros(P + 1, dtype=torch.bool, device=DEV).index_fill_(0, torch.where(slot == 0, page, P), True)
    edge = torch.tensor([-float("inf"), float("inf")], device=DEV).view(1, 1, 2, 1)
    planes = torch.where(start[:P].view(-1, 1, 1, 1), edge, planes)
    at = page.view(-1, 1, 1).expand_as(x)
    top = planes[:, :, 0].contiguous().scatter_reduce_(0, at, x, "amax")
    low = planes[:, :, 1].contiguous().scatter_reduce_(0, at, x, "amin")
    s["planes"].copy_(torch.stack([top, low], 2))
    if c["cache"] != "e2m1":
        return _pools(s)
    return (s["planes"],) + _read(s, s["table"], s["after"], _longest(c))


def _read(s, table, lens, n):
    c = s["case"]
    heads = torch.arange(c["Hk"], device=DEV).view(1, -1, 1)
    pages = table[:, : _pages(n)].clamp(min=0).long().unsqueeze(1)
    live = (torch.arange(n, device=DEV) < lens.unsqueeze(1)).view(c["B"], 1, -1, 1)
    return tuple(torch.where(live, _value(s, name, pages, heads).flatten(2, 3)[:, :, :n], 0.0).to(s["dtype"])
                 for name in ("k", "v"))


def _plain_decode(s):
    c = s["case"]
    B, H, Hk, D = c["B"], c["H"], c["Hk"], c["D"]
    N = s["table"].shape[1] * PAGE
    out = torch.empty(B, 1, Hk, H // Hk, D, dtype=s["dtype"], device=DEV)
    mass = s["mass"].clone() if c["op"] == "mass" else None
    # a KV head at a time: the values of all of them in 32 bits would not fit
    for h in range(Hk):
        pages = s["table"].clamp(min=0).long()
        k, v = (_value(s, name, pages, h).flatten(1, 2) for name in ("k", "v"))          # [B, N, D]
        q = s["q"].reshape(B, Hk, H // Hk, D)[:, h].float().transpose(1, 2).contiguous()
        x = torch.bmm(k, q) * s["scale"]                                                 # [B, N, G]
        x = x.masked_fill((torch.arange(N, device=DEV) >= s["lens"].view(B, 1)).unsqueeze(-1), -float("inf"))
        p = torch.exp(x - x.amax(1, keepdim=True).clamp(min=-1e30))
        total = p.sum(1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
        out[:, 0, h] = torch.bmm(p.transpose(1, 2).contiguous(), v).to(s["dtype"])
        if mass is not None:
            mass[:, h] += p.sum(-1)
    out = out.view(B, 1, H, D)
    return out if mass is None else {"out": out, "mass": mass}


def _plain_evict(s):
    c = s["case"]
    B, Hk, keep = c["B"], c["Hk"], c["keep"]
    N = s["table"].shape[1] * PAGE
    at, n = torch.arange(N, device=DEV), s["lens"].view(B, 1, 1)
    lens = s["lens"].clamp(max=keep)
    forced = (at < c["first"]) | (at >= n - c["recent"])
    order = s["mass"].masked_fill(forced, float("inf")).masked_fill(at >= n, -float("inf"))
    order = order.sort(dim=-1, descending=True, stable=True)[1]
    order = torch.nn.functional.pad(order, (0, max(0, keep - N)), value=N)[..., :keep]
    live = torch.arange(keep, device=DEV) < lens.view(B, 1, 1)
    kept = order.masked_fill(~live, N).sort(-1)[0]                                        # [B, Hk, keep]
    # kept token j of a head goes to slot j of the new pages
    b, h, j = torch.nonzero(live.expand(B, Hk, keep), as_tuple=True)
    src, dst = kept[b, h, j], s["new_table"][b, j // PAGE].long()
    page, slot, to = s["table"][b, src // PAGE].long(), src % PAGE, j % PAGE
    for name in ("k", "v"):
        pages = s[name + "_pages"]
        raw = pages.view(torch.uint8) if c["cache"] == "e4m3" else pages
        raw[dst, h, to] = raw[page, h, slot]
        if c["cache"] == "e4m3":
            s[name + "_scale"][dst, h, to] = s[name + "_scale"][page, h, slot]
        if c["cache"] == "e2m1":
            scale = s[name + "_scale"].transpose(2, 3)
            scale[dst, h, to] = scale[page, h, slot]
    mass = torch.zeros(B, Hk, s["new_table"].shape[1] * PAGE, device=DEV)
    mass[b, h, j] = s["mass"][b, h, src]
    # summaries of the kept keys as they are stored
    heads = torch.arange(Hk, device=DEV).view(1, -1, 1)
    x = _value(s, "k", s["new_table"].clamp(min=0).long().unsqueeze(1), heads)            # [B, Hk, pages, 64, D]
    empty = ~torch.nn.functional.pad(live, (0, x.shape[2] * PAGE - keep)).view(B, 1, -1, PAGE, 1)
    both = torch.stack([x.masked_fill(empty, -float("inf")).amax(3), x.masked_fill(empty, float("inf")).amin(3)], 3)
    b, j = torch.nonzero(~empty[:, 0, :, 0, 0], as_tuple=True)
    s["planes"][s["new_table"][b, j].long()] = both[b, :, j].to(s["dtype"])
    pools = _pools(s) if c["cache"] != "e2m1" else dict(zip(("planes", "k", "v"), (s["planes"],) + _read(
        s, s["new_table"], lens, keep)))
    return {"kept": kept.to(torch.int32), "seq_lens": lens, "mass": mass, **pools}


_PLAIN = {"rotary": _plain_rotary, "write": _plain_write, "decode": _plain_decode, "mass": _plain_decode,
          "evict": _plain_evict}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---- definitions in 64 bits -----------------------------------------------------------------

def _e2m1_of(x, largest):
    """Values of x [..., 32] fp64 held in four bits, by the format's own grid: one bit behind the
    leading one, steps of a half below 2, halves to even; the scale from the largest magnitude."""
    x = x.clamp(-largest, largest)
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -160) / 6))
    e = torch.where(top > 6 * torch.exp2(e), e + 1, e)                # log2's own rounding
    e = torch.where(top <= 6 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top == 0, torch.zeros_like(e), e.clamp(-127, 127))
    y = x * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)
    return torch.round(y / step) * step * torch.exp2(e)


def _turned(c, x, positions):
    """x [..., D] fp64 as complex numbers times exp(i pos f), by the definition of each frequency."""
    r, how = c["rot"], _SCALED[c["scaling"]]
    f, m = [], 1.0
    for j in range(r // 2):
        w = math.exp(-2 * j / r * math.log(10000.0))
        if c["scaling"] == "linear":
            w /= how["factor"]
        if c["scaling"] == "ntk":
            w = (10000.0 * how["factor"] ** (r / (r - 2))) ** (-2 * j / r)
        if c["scaling"] == "yarn":
            def pair(turns):
                return r / 2 * math.log(how["original"] / (2 * math.pi * turns), 10000.0)
            low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), r - 1)
            share = min(max((j - low) / max(high - low, 0.001), 0.0), 1.0)
            w = w + share * (w / how["factor"] - w)
            m = 0.1 * math.log(how["factor"]) + 1
        f.append(w)
    z = x[..., :r].unflatten(-1, (-1, 2)) if c["interleaved"] else x[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
    angle = positions.double().unsqueeze(-1) * torch.tensor(f, dtype=torch.float64, device=DEV)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * torch.polar(torch.full_like(angle, m), angle))
    y = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
    return torch.cat([y, x[..., r:]], -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    B, Hk, D = c["B"], c["Hk"], c["D"]
    if c["op"] == "rotary":
        if not c["grad"]:
            at = s["positions"].unsqueeze(1)
            return _turned(c, s["q"].double(), at), _turned(c, s["k"].double(), at)
        out = [_turned(c, s[name].detach().double(), s["positions"]) for name in ("q", "k")]
        # the gradient of a rotation is the rotation the other way
        return tuple(out) + tuple(_turned(c, s[name].double(), -s["positions"]) for name in ("dq", "dk"))
    n, new = _lengths(c)
    table = s["table"].tolist()

    # the values of sequence b's first tokens for KV head h
    def held(name, b, h, count):
        pages = torch.tensor(table[b][: _pages(count)], device=DEV, dtype=torch.long)
        x = s[name + "_pages"][pages, h]
        if c["cache"] == "e2m1":
            both = torch.stack([x & 15, x >> 4], -1).flatten(-2).double()
            size = both % 8
            x = torch.where(size < 2, size / 2, torch.exp2(torch.floor(size / 2) - 1) * (1 + (size % 2) / 2))
            x = torch.where(both >= 8, -x, x)
            e = s[name + "_scale"][pages, h].double() - 127
            x = x * torch.exp2(e).transpose(1, 2).repeat_interleave(GROUP, -1)
        if c["cache"] == "e4m3":
            x = x.double() * torch.exp2(s[name + "_scale"][pages, h].double() - 127).unsqueeze(-1)
        return x.double().flatten(0, 1)[:count]

    if c["op"] == "write":
        pools = {k: v.double() for k, v in _pools(s).items() if "scale" not in k}
        back = torch.zeros(2, B, Hk, _longest(c), D, dtype=torch.float64, device=DEV)
        at = 0
        for b in range(B):
            pos = torch.arange(n[b], n[b] + new[b], device=DEV)
            page, slot = torch.tensor(table[b], device=DEV)[pos // PAGE], pos % PAGE
            for i, name in enumerate(("k", "v")):
                x = s[name][at : at + new[b]].double()
                if name == "k" and c["turned"]:
                    x = _turned(c, x, s["positions"][at : at + new[b]].unsqueeze(1))
                if name == "k":
                    for p in range(n[b] // PAGE, _pages(n[b] + new[b])):
                        mine = x[max(0, p * PAGE - n[b]) : (p + 1) * PAGE - n[b]]
                        old = pools["planes"][table[b][p]]
                        hi, lo = mine.amax(0), mine.amin(0)
                        if p * PAGE < n[b]:
                            hi, lo = torch.maximum(hi, old[:, 0]), torch.minimum(lo, old[:, 1])
                        pools["planes"][table[b][p]] = torch.stack([hi, lo], 1)
                if c["cache"] == "e2m1":
                    for h in range(Hk):
                        back[i, b, h, : n[b]] = held(name, b, h, n[b])
                    x = _e2m1_of(x.unflatten(-1, (-1, GROUP)), LARGEST[c["dtype"]]).flatten(-2)
                    back[i, b, :, n[b] : n[b] + new[b]] = x.transpose(0, 1)
                else:
                    pools[name + "_pages"][page, :, slot] = x
            at += new[b]
        return (pools["planes"], back[0], back[1]) if c["cache"] == "e2m1" else pools
    if c["op"] == "evict":
        keep, fresh = c["keep"], s["new_table"].tolist()
        out = {k: None if "scale" in k else v.double() for k, v in _pools(s).items()}
        out.update(kept=None, seq_lens=None)
        out["mass"] = torch.zeros(B, Hk, len(fresh[0]) * PAGE, dtype=torch.float64, device=DEV)
        back = torch.zeros(2, B, Hk, keep, D, dtype=torch.float64, device=DEV)
        for b in range(B):
            for h in range(Hk):
                mass = s["mass"][b, h, : n[b]].double()
                free = list(range(c["first"], max(n[b] - c["recent"], c["first"])))
                room = keep - (n[b] - len(free))
                tokens = torch.arange(n[b], device=DEV)
                if n[b] > keep:
                    rank = mass[free[0] : free[-1] + 1].sort(descending=True, stable=True)[1][:room] + free[0]
                    tokens = torch.cat([tokens[: free[0]], rank.sort()[0], tokens[free[-1] + 1 :]])
                m = len(tokens)
                out["mass"][b, h, :m] = mass[tokens]
                values = [held(name, b, h, n[b])[tokens] for name in ("k", "v")]
                for j in range(_pages(m)):
                    part, dst = slice(j * PAGE, min((j + 1) * PAGE, m)), fresh[b][j]
                    out["planes"][dst, h, 0] = values[0][part].amax(0)
                    out["planes"][dst, h, 1] = values[0][part].amin(0)
                    for i, name in enumerate(("k", "v")):
                        back[i, b, h, part] = values[i][part]
                        if c["cache"] == "e2m1":
                            continue
                        src = torch.tensor(table[b], device=DEV)[tokens[part] // PAGE]
                        out[name + "_pages"][dst, h, : part.stop - part.start] = \
                            s[name + "_pages"][src, h, tokens[part] % PAGE].double()
        if c["cache"] == "e2m1":
            out = {k: out[k] for k in ("kept", "seq_lens", "mass", "planes")}
            out.update(k=back[0], v=back[1])
            return out
        return {k: out[k] for k in ("kept", "seq_lens", "mass", *_pools(s))}
    out = torch.zeros(B, 1, c["H"], D, dtype=torch.float64, device=DEV)
    mass = s["mass"].double() if c["op"] == "mass" else None
    G = c["H"] // Hk
    for b in range(B):
        for h in range(Hk if n[b] else 0):
            k, v = held("k", b, h, n[b]), held("v", b, h, n[b])
            q = s["q"][b, h * G : (h + 1) * G, 0].double()
            p = torch.softmax((q @ k.T) * s["scale"], -1)
            out[b, 0, h * G : (h + 1) * G] = p @ v
            if mass is not None:
                mass[b, h, : n[b]] += p.sum(0)
    return out if mass is None else {"out": out, "mass": mass}
