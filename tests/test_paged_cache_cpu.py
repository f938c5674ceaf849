"""The paged cache's argument checks and size queries, which need no GPU."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

import _capi
import paged_cache as pc


def struct(**kw):
    s = dict(k_pages=16, v_pages=16, sk_p=16384, sk_h=8192, sk_n=128, sv_p=16384, sv_h=8192, sv_n=128,
             planes=16, num_pages=4, Hk=2, D=128, dtype=_capi.DTYPE_BF16, cache_dtype=_capi.CACHE_MODEL)
    s.update(kw)
    return _capi.PagedCacheStruct(**s)


def decode(lib, c, B=1, H=4, pages=8, scale=0.1, q=16, kv=None, counts=None, slots=0, out=16, ws=16, n=1 << 30,
           table=16, st=8):
    return lib.ugbsa_paged_decode(ctypes.addressof(c) if c else None, q, 512, 128, 128, 1, H, 16, table, st, B,
                                  pages, scale, kv, counts, slots, out, 512, 128, 1, ws, n, None)


def select(lib, c, k_base=4, k_slots=8, scaling=0.1, tau=0.1, ws=16, n=1 << 30):
    return lib.ugbsa_paged_select(ctypes.addressof(c), 16, 512, 128, 128, 1, 4, 16, 16, 8, 1, 8, scaling, k_base,
                                  k_slots, tau, 16, 16, None, None, ws, n, None)


def refused(lib, rc, code, word):
    assert rc == code and word in lib.ugbsa_last_error().decode(), (rc, lib.ugbsa_last_error())


@pytest.fixture(scope="module")
def lib():
    return _capi.lib()


def test_decode_refusals(lib):
    refused(lib, decode(lib, None), -1, "cache is null")
    refused(lib, decode(lib, struct(D=96)), -1, "head_dim")
    refused(lib, decode(lib, struct(dtype=7)), -3, "dtype")
    refused(lib, decode(lib, struct(cache_dtype=9)), -3, "cache dtype")
    refused(lib, decode(lib, struct(Hk=0)), -1, "positive")
    refused(lib, decode(lib, struct(), H=5), -1, "multiple")
    refused(lib, decode(lib, struct(num_pages=0)), -1, "num_pages")
    refused(lib, decode(lib, struct(), pages=0), -1, "max_pages")
    refused(lib, decode(lib, struct(), pages=(1 << 24) + 1), -1, "max_pages")
    refused(lib, decode(lib, struct(), B=65536), -1, "65535")
    refused(lib, decode(lib, struct(), table=None), -1, "null")
    refused(lib, decode(lib, struct(), st=-8), -2, "stride")
    refused(lib, decode(lib, struct(k_pages=None)), -1, "null")
    refused(lib, decode(lib, struct(k_pages=8)), -2, "aligned")
    refused(lib, decode(lib, struct(sv_n=132)), -2, "aligned")
    refused(lib, decode(lib, struct(cache_dtype=_capi.CACHE_E4M3)), -1, "scale")
    refused(lib, decode(lib, struct(cache_dtype=_capi.CACHE_E4M3, k_scale=16, v_scale=17)), -2, "aligned")
    refused(lib, decode(lib, struct(cache_dtype=_capi.CACHE_E4M3, k_scale=16, v_scale=16, sk_n=136)), -2, "aligned")
    refused(lib, decode(lib, struct(), q=None), -1, "q is null")
    for scale in (float("nan"), float("inf")):
        refused(lib, decode(lib, struct(), scale=scale), -1, "scale")
    refused(lib, decode(lib, struct(), kv=16, slots=0), -1, "k_slots")
    refused(lib, decode(lib, struct(), counts=16), -1, "counts")
    refused(lib, decode(lib, struct(), out=None), -2, "out")
    need = lib.ugbsa_paged_decode_workspace_elems(1, 4, 2, 128, 64, _capi.CACHE_MODEL)
    assert need > 0
    refused(lib, decode(lib, struct(), pages=64, n=need - 1), -1, "workspace")
    refused(lib, decode(lib, struct(), pages=64, ws=None), -1, "workspace")


def test_select_refusals(lib):
    refused(lib, select(lib, struct(planes=None)), -1, "planes")
    refused(lib, select(lib, struct(planes=24)), -1, "planes")
    refused(lib, select(lib, struct(), k_base=2), -1, "k_base")
    refused(lib, select(lib, struct(), k_slots=3), -1, "k_base")
    for scaling in (0.0, -1.0, float("inf"), float("nan")):
        refused(lib, select(lib, struct(), scaling=scaling), -1, "scaling")
    refused(lib, select(lib, struct(), tau=float("nan")), -1, "tau")
    need = lib.ugbsa_paged_select_workspace_elems(1, 2, 8)
    refused(lib, select(lib, struct(), n=need - 1), -1, "workspace")
    refused(lib, select(lib, struct(), ws=20), -2, "workspace")


def test_write_and_read_refusals(lib):
    c = struct()

    def write(T=4, B=1, cu=16, k=16, sk=256):
        return lib.ugbsa_paged_write(ctypes.addressof(c), k, sk, 128, 1, 16, 256, 128, 1, cu, 16, 16, 8, B, T, 8, None)
    refused(lib, write(T=-1), -1, "T=")
    refused(lib, write(T=3, B=4, cu=None), -1, "T=")
    refused(lib, write(k=None), -1, "k is null")
    refused(lib, write(k=18), -2, "aligned")
    refused(lib, write(sk=250), -2, "strides")
    assert write(T=0) == 0                      # nothing to write: no launch

    def read(N=64, out=16, sd=1):
        return lib.ugbsa_paged_read(ctypes.addressof(c), 16, 16, 8, 1, 8, N, out, 8192, 8192, 128, sd,
                                    16, 8192, 8192, 128, 1, None)
    refused(lib, read(N=0), -1, "N must")
    refused(lib, read(N=(1 << 29) + 1), -1, "N must")
    refused(lib, read(out=None), -1, "null")
    refused(lib, read(sd=2), -2, "stride")


def test_workspace_queries_of_sizes_no_call_takes(lib):
    for B, H, Hk, D, units in ((0, 4, 2, 128, 8), (1, 0, 2, 128, 8), (1, 5, 2, 128, 8), (1, 4, 2, 96, 8),
                               (1, 4, 2, 128, 0), (1, 4, 2, 128, -1)):
        assert lib.ugbsa_paged_decode_workspace_elems(B, H, Hk, D, units, _capi.CACHE_E4M3) == 0
    assert lib.ugbsa_paged_select_workspace_elems(0, 2, 8) == lib.ugbsa_paged_select_workspace_elems(1, 2, 0) == 0


def test_caches_of_host_tensors_are_refused():
    pages = torch.zeros(2, 1, 64, 64, dtype=torch.bfloat16)
    for make in (lambda: pc.PagedCache(pages, pages), lambda: pc.PagedCache(pages, None),
                 lambda: pc.PagedCache(pages.float(), pages.float()),
                 lambda: pc.PagedCache(pages[:, :, :32], pages[:, :, :32]),
                 lambda: pc.PagedCache(pages, pages, planes=torch.zeros(2, 1, 2, 32, dtype=torch.bfloat16)),
                 lambda: pc.PagedCache(pages.transpose(2, 3), pages.transpose(2, 3)),
                 lambda: pc.PagedCache.empty(2, 1, 64, torch.bfloat16, "cpu", e4m3=True)):
        with pytest.raises(AssertionError):
            make()


# ---- argument checks of the Python calls, on host tensors ----------------------------------------

def host_cache(dtype=torch.bfloat16, Hk=2, D=64, P=3):
    """What the calls look at of a cache; pages that no call gets as far as reading."""
    pages = torch.zeros(P, Hk, 64, D, dtype=dtype)
    return SimpleNamespace(dtype=dtype, device=torch.device("cpu"), k_pages=pages, v_pages=pages.clone(),
                           planes=torch.zeros(P, Hk, 2, D, dtype=dtype), _call=(None, -1, Hk, D), _writable=True,
                           _struct=SimpleNamespace(cache_dtype=_capi.CACHE_MODEL))


def test_decode_refuses_an_empty_list(monkeypatch):
    """A list of no entries is no call for every page, which is what a null list asks the C side for."""
    def launched(*a):
        raise RuntimeError("launched")
    monkeypatch.setattr(pc, "_launch", launched)
    cache, q = host_cache(), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for shape in ((1, 2, 0), (2,), ()):
        with pytest.raises(AssertionError, match="at least one slot"):
            pc.paged_decode(q, cache, table, lens, 0.1, kv_idx=torch.zeros(shape, dtype=torch.int32))
    lists = torch.zeros(1, 2, 5, dtype=torch.int32)
    with pytest.raises(AssertionError, match="at least one slot"):
        pc.paged_decode(q, cache, table, lens, 0.1, kv_idx=lists[..., :0])
    with pytest.raises(RuntimeError, match="launched"):
        pc.paged_decode(q, cache, table, lens, 0.1, kv_idx=lists[..., :1].contiguous())


def calls(cache, q, k, v, out=None, pair=None):
    """Each operator once on the tensors given."""
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    return {"decode": lambda: pc.paged_decode(q, cache, table, lens, 0.1, out=out),
            "select": lambda: pc.paged_select(q, cache, table, lens, 0.1, 3, 4),
            "write": lambda: pc.paged_write(cache, k, v, table, lens),
            "read": lambda: pc.paged_read(cache, table, lens, 5, out=pair)}


def no_launch(monkeypatch):
    monkeypatch.setattr(pc, "_launch", lambda *a: None)


@pytest.mark.filterwarnings("ignore")
def test_tangents_and_traces_are_refused(monkeypatch):
    """A dual tensor requires no gradient and points at its primal: its tangent would be dropped."""
    no_launch(monkeypatch)
    fw = torch.autograd.forward_ad
    q, k = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    out, pair = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16), [torch.zeros(1, 2, 5, 64, dtype=torch.bfloat16) for _ in "kv"]
    with fw.dual_level():
        def dual(t):
            return fw.make_dual(t, torch.ones_like(t))
        for name, args in (("decode", (dual(q), k, k)), ("select", (dual(q), k, k)), ("write", (q, dual(k), k)),
                           ("write", (q, k, dual(k))), ("decode", (q, k, k, dual(out))),
                           ("read", (q, k, k, None, (pair[0], dual(pair[1]))))):
            with pytest.raises(AssertionError, match="forward-mode"):
                calls(host_cache(), *args)[name]()
        for call in calls(host_cache(), q, k, k, out, pair).values():        # no tangent in reach
            call()
    for name in ("decode", "select", "write", "read"):
        def traced(x, name=name):
            calls(host_cache(), q + x, k + x, k + x)[name]()
            return x
        with pytest.raises(AssertionError, match="traced"):
            torch.jit.trace(traced, torch.zeros(1, dtype=torch.bfloat16), check_trace=False)


def test_outputs_that_do_not_hold_what_is_stored_are_refused(monkeypatch):
    """Negated views, tensors that record gradients, elements that share memory, K and V in one place."""
    no_launch(monkeypatch)
    bf = torch.bfloat16
    q, k = torch.zeros(1, 4, 1, 64, dtype=bf), torch.zeros(1, 2, 64, dtype=bf)
    for bad in (torch._neg_view(torch.zeros(1, 1, 4, 64, dtype=bf)), torch.zeros(1, 1, 4, 64, dtype=bf, requires_grad=True),
                torch.zeros(1, 1, 1, 64, dtype=bf).expand(1, 1, 4, 64), torch.zeros(1, 1, 4, 128, dtype=bf)):
        with pytest.raises(AssertionError, match="out"):
            calls(host_cache(), q, k, k, out=bad)["decode"]()
    good = torch.zeros(1, 2, 5, 64, dtype=bf)
    for bad in (torch._neg_view(good.clone()), good.clone().requires_grad_(),
                torch.zeros(1, 1, 5, 64, dtype=bf).expand(1, 2, 5, 64), good):
        for pair in ((good, bad), (bad, good)):
            with pytest.raises(AssertionError, match="out"):
                calls(host_cache(), q, k, k, pair=pair)["read"]()
    with torch.no_grad():                                  # as for any in-place write
        calls(host_cache(), q, k, k, out=torch.zeros(1, 1, 4, 64, dtype=bf, requires_grad=True))["decode"]()
    calls(host_cache(), q, k, k, out=torch.zeros(4, 1, 1, 64, dtype=bf).transpose(0, 2))["decode"]()
    calls(host_cache(), q, k, k, pair=(good, torch.zeros(2, 1, 5, 64, dtype=bf).transpose(0, 1)))["read"]()


def test_operands_that_cannot_be_read_in_place_are_copied():
    """Also those that count as contiguous: at an odd address, or with an odd stride of a dimension of
    one element (the query or the one new token of a batch of one, cut out of a wider projection)."""
    bf, cache = torch.bfloat16, host_cache()
    flat = torch.arange(4096, dtype=torch.float32).to(bf)
    views = [flat[4:4 + 256].view(1, 4, 1, 64),                               # 8 bytes past a boundary
             flat[:258 * 2].view(2, 258)[:1, :256].view(1, 1, 4, 64).transpose(1, 2)[:1],
             flat[:257].view(1, 257)[:, :256].view(1, 4, 1, 64),              # batch stride 257
             flat[:4 * 65].view(1, 4, 1, 65)[..., :64], flat[:256].view(1, 64, 1, 4).transpose(1, 3)]
    for v in views:
        t = pc._operand("q", v, cache, (1, 4, 1, 64))
        assert torch.equal(t, v) and t.data_ptr() % 16 == 0 and t.stride(-1) == 1
        assert not any(s % 8 for s in t.stride()[:-1]), v.stride()
    k = flat[:131].view(1, 131)[:, :128].view(1, 2, 64)
    t = pc._operand("k", k, cache, (1, 2, 64))
    assert torch.equal(t, k) and not any(s % 8 for s in t.stride()[:-1])
    same = flat[:256].view(1, 4, 1, 64)
    assert pc._operand("q", same, cache, (1, 4, 1, 64)) is same
