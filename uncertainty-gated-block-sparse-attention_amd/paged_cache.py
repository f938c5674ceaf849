"""Paged key-value cache for serving: written, read back, selected from and decoded over.

The dispatcher's decode attends to a contiguous ``[B, Hk, N, D]`` cache; a server keeps keys and
values in pages of 64 tokens, the selection block, that a block table names.  Pages hold the
model's dtype, e4m3 codes with a power-of-two scale per token and head, or e2m1 codes (four bits) with one per
32 dims of it, and beside them stands each page's Quest summary (K-max, K-min of the keys as given,
before they are rounded to codes), kept up to date as tokens are written:

    cache = PagedCache.empty(num_pages, Hk, D, torch.bfloat16, "cuda", e4m3=True)
    paged_write(cache, k, v, block_table, seq_lens, cu_new=cu)     # prompts [T, Hk, D], packed
    ...                                                            # per generated token:
    paged_write(cache, k1, v1, block_table, seq_lens)              # [B, Hk, D], one token each
    seq_lens += 1
    sel = paged_select(q, cache, block_table, seq_lens, scale, k_base=64, k_slots=128, tau=0.01)
    out = paged_decode(q, cache, block_table, seq_lens, scale, sel.kv_idx, sel.counts)
    k, v = paged_read(cache, block_table, seq_lens, N)             # [B, Hk, N, D], contiguous

A cache that has to stay within its pages follows the attention weights of its tokens
(``paged_decode(..., mass=)``) and is cut back to the heaviest by ``paged_evict``; keys can be turned by
their positions on the way in (``paged_write(..., rotary=, positions=)``).

``block_table`` [B, max_pages] int32 and ``seq_lens`` [B] int32 live on the device: no call reads
them on the host, and every call is asynchronous on the current stream and can be captured in a
graph.  Lengths outside [0, 64 * max_pages] are taken as the nearer end; table entries outside the
cache name absent pages, which are never written, read as zeros and take no part in attention.

The operators have no derivatives: tensors that require gradients are refused where gradients are
recorded, and so are tensors with a forward-mode tangent and calls that are being traced.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field

import torch
from torch.autograd import forward_ad

import _capi

PAGE = 64    # tokens per page: the selection block
GROUP = 32   # dims of a token's head that share an e2m1 scale

_tracing_state = torch._C._get_tracing_state


@dataclass(frozen=True, eq=False)
class PagedCache:
    """Pages of one layer and their summaries.  The handle keeps the tensors and their addresses:
    they are written in place, never resized or pointed elsewhere.

    k_pages, v_pages : [P, Hk, 64, D] in ``dtype`` or ``torch.float8_e4m3fn``, or [P, Hk, 64, D / 2] uint8,
    two e2m1 codes a byte, the even dim in its low four bits (unit stride on head_dim, 16-byte aligned
    rows, any other strides; expanded pages, or one tensor for both, can be read but not written)
    k_scale, v_scale : uint8 contiguous, [P, Hk, 64] for e4m3 pages, [P, Hk, D / 32, 64] for e2m1: a value
    is code * 2^(byte - 127) (e2m1: NaN where the byte is 255)
    planes : [P, Hk, 2, D] in ``dtype``, contiguous: K-max and K-min of each page.  Optional where
    nothing is selected; a cache of planes alone (no pages) serves ``paged_select`` only.
    dtype : bf16 or fp16, the format of q, k, v and of every result
    """

    k_pages: torch.Tensor | None
    v_pages: torch.Tensor | None
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None
    planes: torch.Tensor | None = None
    dtype: torch.dtype | None = None
    device: torch.device = field(init=False, default=None)
    _struct: _capi.PagedCacheStruct = field(init=False, repr=False, compare=False, default=None)
    _call: tuple = field(init=False, repr=False, compare=False, default=None)   # address, device, Hk, D
    _writable: bool = field(init=False, repr=False, compare=False, default=False)

    def __post_init__(self):
        k, v, planes = self.k_pages, self.v_pages, self.planes
        assert (k is None) == (v is None), "k_pages and v_pages go together"
        assert k is not None or planes is not None, "pages or planes required"
        dtype = self.dtype
        e4m3 = k is not None and k.dtype == torch.float8_e4m3fn
        e2m1 = k is not None and k.dtype == torch.uint8
        codes = e4m3 or e2m1
        if dtype is None:
            assert not codes or planes is not None, "dtype required (codes do not tell it)"
            dtype = planes.dtype if planes is not None else k.dtype
            object.__setattr__(self, "dtype", dtype)
        code = _capi.dtype_code(dtype)
        s = _capi.PagedCacheStruct(dtype=code,
                                   cache_dtype=_capi.CACHE_E2M1 if e2m1 else _capi.CACHE_E4M3 if e4m3
                                   else _capi.CACHE_MODEL)
        if k is not None:
            assert k.dim() == 4 and k.shape == v.shape and k.shape[2] == PAGE, "pages [P, Hk, 64, D] expected"
            assert k.dtype == v.dtype and (codes or k.dtype == dtype), f"pages: {dtype}, e4m3 or uint8 required"
            s.num_pages, s.Hk, _, s.D = k.shape
            s.D *= 2 if e2m1 else 1
            unit = 16 // k.element_size()
            for t in (k, v):
                assert t.stride(3) == 1 and t.data_ptr() % 16 == 0 and not any(x % unit for x in t.stride()[:3]), \
                    "pages need unit head_dim stride and 16-byte aligned rows"
            s.k_pages, s.v_pages = k.data_ptr(), v.data_ptr()
            s.sk_p, s.sk_h, s.sk_n, _ = k.stride()
            s.sv_p, s.sv_h, s.sv_n, _ = v.stride()
            assert codes == (self.k_scale is not None) == (self.v_scale is not None), \
                "scales go with quantised pages"
            if codes:
                want = (s.num_pages, s.Hk, s.D // GROUP, PAGE) if e2m1 else (s.num_pages, s.Hk, PAGE)
                for t in (self.k_scale, self.v_scale):
                    assert t.shape == want and t.dtype == torch.uint8 and t.is_contiguous() \
                        and t.data_ptr() % (16 if e2m1 else 8) == 0, f"scales {list(want)} uint8 contiguous expected"
                s.k_scale, s.v_scale = self.k_scale.data_ptr(), self.v_scale.data_ptr()
        if planes is not None:
            if k is None:
                assert planes.dim() == 4, "planes [P, Hk, 2, D] expected"
                s.num_pages, s.Hk, _, s.D = planes.shape
            assert tuple(planes.shape) == (s.num_pages, s.Hk, 2, s.D) and planes.dtype == dtype \
                and planes.is_contiguous() and planes.data_ptr() % 16 == 0, "planes [P, Hk, 2, D] expected"
            s.planes = planes.data_ptr()
        assert s.D in (64, 128, 256), f"head_dim {s.D} not supported (64, 128, 256)"
        tensors = [t for t in (k, v, self.k_scale, self.v_scale, planes) if t is not None]
        assert all(t.is_cuda and t.device == tensors[0].device for t in tensors), "HIP tensors of one device required"
        assert not any(t.requires_grad or t.is_neg() for t in tensors), "plain tensors without gradients required"
        _check_unwatched(*tensors)
        object.__setattr__(self, "_writable", k is not None and k.data_ptr() != v.data_ptr() and not any(
            st == 0 and n > 1 for t in (k, v) for st, n in zip(t.stride(), t.shape)))
        object.__setattr__(self, "_struct", s)
        object.__setattr__(self, "device", tensors[0].device)
        object.__setattr__(self, "_call", (ctypes.addressof(s), tensors[0].get_device(), s.Hk, s.D))

    @classmethod
    def empty(cls, num_pages, Hk, D, dtype, device, e4m3=False, summaries=True, e2m1=False):
        """Uninitialised pages: every slot a sequence reads is written first."""
        assert not (e4m3 and e2m1), "pages are e4m3 or e2m1"
        shape = (num_pages, Hk, PAGE, D // 2 if e2m1 else D)
        pages = torch.uint8 if e2m1 else torch.float8_e4m3fn if e4m3 else dtype
        scales = (num_pages, Hk, D // GROUP, PAGE) if e2m1 else shape[:3]
        k, v = (torch.empty(shape, dtype=pages, device=device) for _ in range(2))
        ks, vs = (torch.empty(scales, dtype=torch.uint8, device=device) if e4m3 or e2m1 else None for _ in range(2))
        planes = torch.empty(num_pages, Hk, 2, D, dtype=dtype, device=device) if summaries else None
        return cls(k, v, ks, vs, planes, dtype)


@dataclass
class PagedSelection:
    kv_idx: torch.Tensor       # int32 [B, Hk, k_slots] ascending pages of the sequence, then max_pages
    counts: torch.Tensor       # int32 [B, Hk] pages listed
    sigma: torch.Tensor        # fp32 [B, Hk] margin at the cut
    uncertain: torch.Tensor    # uint8 [B, Hk]


def _check_unwatched(*tensors):
    """Refuses what would lose or freeze values without an error: a tangent beside a tensor's data, a
    trace that records the calls around a launch.  (Functional transforms have no data to point at.)"""
    assert _tracing_state() is None, "the paged operators cannot be traced"
    if forward_ad._current_level >= 0:
        assert all(forward_ad.unpack_dual(t).tangent is None for t in tensors
                   if t is not None and t.is_floating_point()), \
            "the paged operators have no forward-mode derivative"


def _watched():
    """Whether a call has to look closer: next to nothing of its time otherwise."""
    return forward_ad._current_level >= 0 or _tracing_state() is not None


def _operand(name, t, cache, shape):
    """A 16-bit tensor of the cache's dtype and device that the kernels read in place."""
    st = t.stride()
    if (t.dtype is cache.dtype and t.get_device() == cache._call[1] and t.shape == shape and st[-1] == 1
            and not (t.requires_grad or t.data_ptr() & 15 or t.is_neg())
            and not any(s & 7 for s in st[:-1])):
        return t
    assert t.dtype == cache.dtype, f"{name}: {cache.dtype} required, got {t.dtype}"
    assert t.device == cache.device, f"{name} must be on the cache's device"
    assert tuple(t.shape) == shape, f"{name} {list(shape)} expected, got {list(t.shape)}"
    assert not (t.requires_grad and torch.is_grad_enabled()), "the paged operators have no backward pass"
    if t.is_neg():
        t = t.resolve_neg()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:-1]):
        # not contiguous(): that is the tensor itself where only the address or the stride of a
        # dimension of one element is in the way
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _check_out(t, cache, shape):
    """A result tensor that the kernels fill in place: what is stored is what the tensor holds, and each
    element has a place of its own."""
    assert t.shape == shape and t.dtype is cache.dtype and t.get_device() == cache._call[1], \
        f"out: {list(shape)} in {cache.dtype} on the cache's device expected"
    assert not t.is_neg() and not (t.requires_grad and torch.is_grad_enabled()), \
        "out: a plain tensor without gradients required"
    assert not any(s == 0 and n > 1 for s, n in zip(t.stride(), shape)), "out: elements share memory"


def _check_ints(name, t, cache, shape):
    assert t.dtype is torch.int32 and t.shape == shape and t.is_contiguous() \
        and t.get_device() == cache._call[1], \
        f"{name} {list(shape)} int32 contiguous on the cache's device expected"


def _table(cache, block_table, seq_lens):
    """(B, max_pages, row stride) of a call's table, whose lengths are checked too."""
    assert block_table.dim() == 2 and block_table.dtype is torch.int32 \
        and block_table.get_device() == cache._call[1], "block_table [B, max_pages] int32 on the cache's device expected"
    B, max_pages = block_table.shape
    st_b, st_p = block_table.stride()
    assert B >= 1 and max_pages >= 1, "block_table is empty"
    assert st_p == 1 or max_pages == 1, "block_table: a row's entries must be contiguous"
    _check_ints("seq_lens", seq_lens, cache, (B,))
    return B, max_pages, st_b


def _launch(cache, what, fn, *args):
    """fn(cache, *args, stream) on the cache's device."""
    address, index, _, _ = cache._call
    if torch._C._cuda_getDevice() == index:
        rc = fn(address, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(address, *args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _capi.check(rc, what)


def paged_write(cache, k, v, block_table, seq_lens, cu_new=None, rotary=None, positions=None):
    """New tokens into the cache, quantised if it holds codes, and its page summaries.

    k, v : [T, Hk, D], the new tokens of all sequences, packed
    cu_new : [B + 1] int32, ascending: sequence b's are rows cu_new[b] .. cu_new[b + 1] - 1; None:
    one token each, row b
    seq_lens : tokens cached before this call; the new ones follow them (the caller adds them up)
    rotary : a ``rotary.Rotary``: keys are turned by ``positions`` [T] int32 on the way, to the bits that
    ``rotary.rotary`` gives; without positions by their places in their sequences

    Rows behind the last sequence and tokens past the table are left out.  Two sequences may share
    pages, but no page that a call writes to may be named twice by the entries it writes through.
    """
    assert cache.k_pages is not None, "a cache of planes alone has no pages"
    assert cache._writable, "pages whose elements share memory cannot be written"
    B, max_pages, st_b = _table(cache, block_table, seq_lens)
    shape = (k.shape[0], *cache._call[2:])
    k = _operand("k", k, cache, shape)
    v = _operand("v", v, cache, shape)
    if _watched():
        _check_unwatched(k, v)
    if cu_new is not None:
        _check_ints("cu_new", cu_new, cache, (B + 1,))
    fn, turn = _capi.lib().ugbsa_paged_write, ()
    if rotary is not None:
        address, index, dims = rotary._call
        assert index == cache._call[1], "rotary must be on the cache's device"
        assert dims <= shape[2], f"rotary: head_dim {shape[2]} must hold the table's {dims} dims"
        if positions is not None:
            _check_ints("positions", positions, cache, (shape[0],))
        fn, turn = _capi.lib().ugbsa_paged_write_rotary, (address, _capi.ptr(positions))
    else:
        assert positions is None, "positions without rotary"
    _launch(cache, "paged_write", fn, k.data_ptr(), *k.stride(),
            v.data_ptr(), *v.stride(), None if cu_new is None else cu_new.data_ptr(), seq_lens.data_ptr(),
            block_table.data_ptr(), st_b, B, shape[0], max_pages, *turn)


def paged_read(cache, block_table, seq_lens, n, out=None):
    """(k, v) [B, Hk, n, D] in ``cache.dtype``: the first n >= 1 cached tokens of every sequence, zeros
    past its length (``out``: a pair of such tensors to fill).  The layout of a contiguous cache, which
    the dispatcher's decode attends to; its sparse prefills take as many queries as keys and so no
    cached prefix."""
    assert cache.k_pages is not None, "a cache of planes alone has no pages"
    B, max_pages, st_b = _table(cache, block_table, seq_lens)
    _, _, Hk, D = cache._call
    shape = (B, Hk, n, D)
    if _watched():
        _check_unwatched(*(() if out is None else out))
    if out is None:
        k, v = (torch.empty(shape, dtype=cache.dtype, device=cache.device) for _ in range(2))
    else:
        k, v = out
        _check_out(k, cache, shape)
        _check_out(v, cache, shape)
        assert k.data_ptr() != v.data_ptr(), "out: k and v are the same memory"
    _launch(cache, "paged_read", _capi.lib().ugbsa_paged_read, seq_lens.data_ptr(), block_table.data_ptr(),
            st_b, B, max_pages, n, k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride())
    return k, v


def paged_select(q, cache, block_table, seq_lens, scaling, k_base, k_slots, tau=0.0):
    """The pages one new token attends to, per sequence and KV head: the decode counterpart of the
    v2 selector.

    q : [B, H, 1, D]; seq_lens counts the new token.  A page's score is the Quest bound of its
    summary, maximised over the KV head's query heads and summed in fp64.  The first and the last
    page are kept, and the best others by (score desc, page asc) up to ``k_base`` >= 3 pages, or
    ``k_slots`` where the margin at the cut, sigma = clamp((s(k) - s(k + 1)) / max(s(1) - s(k + 1),
    1e-9), 0, 2) over the scaled scores of the others, k = k_base - 2, is below ``tau``
    (``Selector.router_tau``'s role; 0 keeps k_base throughout).  A sequence's list depends on no
    other sequence of the batch.  Returns a ``PagedSelection`` for ``paged_decode``.
    """
    assert cache.planes is not None, "the cache keeps no page summaries"
    B, max_pages, st_b = _table(cache, block_table, seq_lens)
    _, _, Hk, D = cache._call
    H = q.shape[1] if q.dim() == 4 else 0
    q = _operand("q", q, cache, (B, H, 1, D))
    if _watched():
        _check_unwatched(q)
    device = cache.device
    kv_idx = torch.empty((B, Hk, max(k_slots, 0)), dtype=torch.int32, device=device)
    counts = torch.empty((B, Hk), dtype=torch.int32, device=device)
    sigma = torch.empty((B, Hk), dtype=torch.float32, device=device)
    uncertain = torch.empty((B, Hk), dtype=torch.uint8, device=device)
    lib = _capi.lib()
    n = lib.ugbsa_paged_select_workspace_elems(B, Hk, max_pages) if max_pages > k_base else 0
    ws = torch.empty(n, dtype=torch.float32, device=device) if n else None
    _launch(cache, "paged_select", lib.ugbsa_paged_select, q.data_ptr(), *q.stride(), H, seq_lens.data_ptr(),
            block_table.data_ptr(), st_b, B, max_pages, scaling, k_base, k_slots, tau, kv_idx.data_ptr(),
            counts.data_ptr(), sigma.data_ptr(), uncertain.data_ptr(), _capi.ptr(ws), n)
    return PagedSelection(kv_idx, counts, sigma, uncertain)


def _check_mass(name, t, cache, shape):
    """Strides (b, h) of weights [B, Hk, >= 64 * pages] fp32 that a call reads or adds to in place."""
    B, Hk, n = shape
    size = t.shape
    assert len(size) == 3 and size[0] == B and size[1] == Hk and size[2] >= n and t.dtype is torch.float32 \
        and t.get_device() == cache._call[1], f"{name} [{B}, {Hk}, >= {n}] fp32 on the cache's device expected"
    st_b, st_h, st_n = t.stride()
    st_b, st_h = st_b if B > 1 else 0, st_h if Hk > 1 else 0      # of one element any will do
    assert st_n == 1 and not (t.data_ptr() & 15 or st_b & 3 or st_h & 3), \
        f"{name}: contiguous, 16-byte aligned rows required"
    assert not (t.is_neg() or t.requires_grad), f"{name}: a plain tensor without gradients required"
    return st_b, st_h


def paged_decode(q, cache, block_table, seq_lens, scale, kv_idx=None, counts=None, out=None, mass=None):
    """Attention of one new token per sequence over its cached tokens, of every page or of the
    listed ones.

    q : [B, H, 1, D]; seq_lens counts the new token, which ``paged_write`` has put in the cache
    kv_idx : [B, Hk, k_slots >= 1] int32, the pages (numbered within the sequence, each at most once)
    that the KV head's query heads attend to; counts [B, Hk] int32: how many entries count (None:
    all).  Entries that are no page of the sequence are skipped.
    mass : [B, Hk, >= 64 * max_pages] fp32, what each cached token's weight adds up to, for ``paged_evict``:
    entry i of a row grows by the sum over the KV head's query heads of token i's softmax weight.  The
    call then keeps its scores meanwhile, B * H * 64 * (max_pages or k_slots) fp32 whatever the lengths are
    Returns [B, 1, H, D] contiguous, the dispatcher's layout (``out`` if given).  A sequence without
    a key gives zeros.  Weights are rounded to ``dtype`` before the product with V.  The launch,
    and the scores' memory with ``mass``, are shaped by the table's (or list's) width: pass a table cut to the
    longest sequence where the batch is short.
    """
    assert cache.k_pages is not None, "a cache of planes alone has no pages"
    B, max_pages, st_b = _table(cache, block_table, seq_lens)
    _, _, Hk, D = cache._call
    H = q.shape[1] if q.dim() == 4 else 0
    q = _operand("q", q, cache, (B, H, 1, D))
    if _watched():
        _check_unwatched(q, out, mass)
    slots = 0
    if kv_idx is not None:
        slots = kv_idx.shape[-1] if kv_idx.dim() == 3 else 0
        assert slots >= 1, "kv_idx [B, Hk, k_slots] with at least one slot expected (counts of 0 list no page)"
        _check_ints("kv_idx", kv_idx, cache, (B, Hk, slots))
    if counts is not None:
        _check_ints("counts", counts, cache, (B, Hk))
    if out is None:
        out = torch.empty((B, 1, H, D), dtype=cache.dtype, device=cache.device)
    else:
        _check_out(out, cache, (B, 1, H, D))
    so_b, _, so_h, so_d = out.stride()
    lib = _capi.lib()
    if mass is not None:
        sm_b, sm_h = _check_mass("mass", mass, cache, (B, Hk, PAGE * max_pages))
        outer, inner = (sm_b, sm_h * (Hk - 1)) if sm_b > sm_h else (sm_h, sm_b * (B - 1))
        assert (B == 1 or sm_b >= mass.shape[2]) and (Hk == 1 or sm_h >= mass.shape[2]) and (
            B == 1 or Hk == 1 or outer >= inner + mass.shape[2]), "mass: rows share memory"
        n = lib.ugbsa_paged_decode_mass_workspace_elems(B, H, Hk, D, slots or max_pages, cache._struct.cache_dtype)
        ws = torch.empty(n, dtype=torch.float32, device=cache.device)
        if not mass.is_inference():       # those have no version for autograd to look at
            torch.autograd.graph.increment_version(mass)
        _launch(cache, "paged_decode_mass", lib.ugbsa_paged_decode_mass, q.data_ptr(), *q.stride(), H,
                seq_lens.data_ptr(), block_table.data_ptr(), st_b, B, max_pages, scale, _capi.ptr(kv_idx),
                _capi.ptr(counts), slots, mass.data_ptr(), sm_b, sm_h, out.data_ptr(), so_b, so_h, so_d,
                ws.data_ptr(), n)
        return out
    n = lib.ugbsa_paged_decode_workspace_elems(B, H, Hk, D, slots or max_pages, cache._struct.cache_dtype)
    ws = torch.empty(n, dtype=torch.float32, device=cache.device) if n else None
    _launch(cache, "paged_decode", lib.ugbsa_paged_decode, q.data_ptr(), *q.stride(), H, seq_lens.data_ptr(),
            block_table.data_ptr(), st_b, B, max_pages, scale, _capi.ptr(kv_idx), _capi.ptr(counts), slots,
            out.data_ptr(), so_b, so_h, so_d, _capi.ptr(ws), n)
    return out


@dataclass
class PagedEviction:
    kept: torch.Tensor         # int32 [B, Hk, keep] tokens that stayed, ascending, then 64 * max_pages
    seq_lens: torch.Tensor     # int32 [B] tokens of each sequence now
    mass: torch.Tensor         # fp32 [B, Hk, 64 * new_pages] their weights, then zeros


def paged_evict(cache, mass, block_table, seq_lens, new_table, keep, recent=0, first=0):
    """Sequences cut back to ``keep`` tokens, packed into other pages: each KV head keeps the first
    ``first`` tokens, the newest ``recent`` and, of the others, those of the largest ``mass``.

    mass : [B, Hk, >= 64 * max_pages] fp32 as ``paged_decode`` adds it up.  Ties stay by the lower token,
    NaN before numbers; tokens of absent pages do not stay
    new_table : [B, new_pages] int32, 64 * new_pages >= keep: the pages that take the kept tokens, in
    their order.  None may be a page that the call reads (those are free afterwards, unless another
    sequence shares them), nor be named twice

    A sequence of no more than ``keep`` tokens keeps all of them (call with the rows of ``block_table``
    that are to be cut back).  Codes and scales are copied as they are; page summaries become those of
    the keys as stored.  Keys keep the positions that turned them: pass later tokens' positions to
    ``rotary`` and ``paged_write``, whose lengths are shorter now.  Returns a ``PagedEviction``.
    """
    assert cache.k_pages is not None, "a cache of planes alone has no pages"
    assert cache._writable, "pages whose elements share memory cannot be written"
    B, max_pages, st_b = _table(cache, block_table, seq_lens)
    _, _, Hk, _ = cache._call
    assert new_table.dim() == 2 and new_table.shape[0] == B and new_table.dtype is torch.int32 \
        and new_table.get_device() == cache._call[1] and new_table.shape[1] >= 1, \
        "new_table [B, new_pages] int32 on the cache's device expected"
    new_pages = new_table.shape[1]
    assert new_table.stride(1) == 1 or new_pages == 1, "new_table: a row's entries must be contiguous"
    sm_b, sm_h = _check_mass("mass", mass, cache, (B, Hk, PAGE * max_pages))
    if _watched():
        _check_unwatched(mass)
    device = cache.device
    kept = torch.empty((B, Hk, max(keep, 0)), dtype=torch.int32, device=device)
    lens = torch.empty(B, dtype=torch.int32, device=device)
    new_mass = torch.empty((B, Hk, PAGE * new_pages), dtype=torch.float32, device=device)
    lib = _capi.lib()
    n = lib.ugbsa_paged_evict_workspace_elems(B, Hk, max_pages)
    ws = torch.empty(n, dtype=torch.float32, device=device) if n else None
    _launch(cache, "paged_evict", lib.ugbsa_paged_evict, mass.data_ptr(), sm_b, sm_h, seq_lens.data_ptr(),
            block_table.data_ptr(), st_b, B, max_pages, new_table.data_ptr(), new_table.stride(0), new_pages, keep,
            recent, first, kept.data_ptr(), lens.data_ptr(), new_mass.data_ptr(), *new_mass.stride()[:2],
            _capi.ptr(ws), n)
    return PagedEviction(kept, lens, new_mass)
