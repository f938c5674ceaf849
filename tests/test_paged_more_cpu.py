"""Argument checks of the four-bit cache, of followed weights and of eviction, which need no GPU."""

import ctypes

import pytest
import torch

import _capi
import paged_cache as pc
from test_paged_cache_cpu import host_cache, refused, struct


@pytest.fixture(scope="module")
def lib():
    return _capi.lib()


def four(**kw):
    s = dict(sk_p=8192, sk_h=4096, sk_n=64, sv_p=8192, sv_h=4096, sv_n=64, k_scale=16, v_scale=16,
             cache_dtype=_capi.CACHE_E2M1)
    s.update(kw)
    return struct(**s)


def mass_call(lib, c, B=1, H=4, pages=8, mass=16, sm_b=1024, sm_h=512, kv=None, slots=0, ws=16, n=1 << 40, out=16):
    return lib.ugbsa_paged_decode_mass(ctypes.addressof(c) if c else None, 16, 512, 128, 128, 1, H, 16, 16, 8, B, pages,
                                       0.1, kv, None, slots, mass, sm_b, sm_h, out, 512, 128, 1, ws, n, None)


def evict_call(lib, c, mass=16, sm=512, lens=16, table=16, new=16, sn=4, pages=4, keep=100, recent=0, first=0, kept=16,
               new_lens=16, new_mass=16, so=256, max_pages=8, ws=None, n=0):
    return lib.ugbsa_paged_evict(ctypes.addressof(c) if c else None, mass, sm, sm, lens, table, 8, 1, max_pages, new, sn,
                                 pages, keep, recent, first, kept, new_lens, new_mass, so, so, ws, n, None)


def test_four_bit_caches(lib):
    for bad, code, word in ((four(k_scale=None), -1, "scale"), (four(v_scale=12), -2, "aligned"),
                            (four(sk_n=72), -2, "aligned"), (four(k_pages=24), -2, "aligned"), (four(D=96), -1, "head_dim"),
                            (four(cache_dtype=3), -3, "cache dtype")):
        refused(lib, mass_call(lib, bad), code, word)
        refused(lib, evict_call(lib, bad), code, word)
    for query in (lib.ugbsa_paged_decode_workspace_elems, lib.ugbsa_paged_decode_mass_workspace_elems):
        assert query(1, 5, 2, 128, 8, _capi.CACHE_E2M1) == query(1, 4, 2, 96, 8, _capi.CACHE_E2M1) == 0
        assert query(1, 4, 2, 128, 0, _capi.CACHE_E2M1) == 0
        assert query(1, 4, 2, 128, 4096, _capi.CACHE_E2M1) > 0


def test_mass_refusals(lib):
    refused(lib, mass_call(lib, None), -1, "cache is null")
    for kw, code, word in ((dict(mass=None), -1, "mass is null"), (dict(mass=8), -2, "mass"), (dict(sm_b=2), -2, "mass"),
                           (dict(sm_h=-4), -2, "mass"), (dict(H=5), -1, "multiple"), (dict(kv=16), -1, "k_slots"),
                           (dict(out=None), -2, "out"), (dict(ws=None), -1, "workspace"), (dict(pages=0), -1, "max_pages"),
                           (dict(B=60000, pages=1 << 20), -1, "2^30")):
        refused(lib, mass_call(lib, four(), **kw), code, word)
    need = lib.ugbsa_paged_decode_mass_workspace_elems(1, 4, 2, 128, 8, _capi.CACHE_E2M1)
    assert need >= 4 * 8 * 64                               # the scores of every head, also where rows are whole
    refused(lib, mass_call(lib, four(), n=need - 1), -1, "workspace")
    refused(lib, mass_call(lib, four(), ws=24), -2, "workspace")


def test_evict_refusals(lib):
    refused(lib, evict_call(lib, None), -1, "cache is null")
    for kw, code, word in ((dict(mass=None), -1, "mass is null"), (dict(mass=4), -2, "mass"), (dict(sm=6), -2, "mass"),
                           (dict(new_mass=None), -1, "new_mass"), (dict(so=2), -2, "new_mass"), (dict(new=None), -1, "null"),
                           (dict(kept=None), -1, "null"), (dict(new_lens=None), -1, "null"), (dict(lens=None), -1, "null"),
                           (dict(table=None), -1, "null"), (dict(sn=-1), -2, "stride"), (dict(pages=0), -1, "new_pages"),
                           (dict(pages=(1 << 24) + 1), -1, "new_pages"), (dict(keep=0), -1, "keep"),
                           (dict(keep=257), -1, "keep"), (dict(recent=-1), -1, "recent"), (dict(first=-1), -1, "recent"),
                           (dict(recent=60, first=41), -1, "recent"), (dict(recent=(1 << 31) - 1, first=(1 << 31) - 1), -1, "recent")):
        refused(lib, evict_call(lib, four(), **kw), code, word)
    assert lib.ugbsa_paged_evict_workspace_elems(1, 2, 8) == lib.ugbsa_paged_evict_workspace_elems(1, 2, 0) == 0
    assert lib.ugbsa_paged_evict_workspace_elems(1, 2, (1 << 24) + 1) == 0
    need = lib.ugbsa_paged_evict_workspace_elems(1, 2, 512)
    assert need > 0
    for kw, code in ((dict(ws=None, n=need), -1), (dict(ws=16, n=need - 1), -1), (dict(ws=8, n=need), -2)):
        refused(lib, evict_call(lib, four(), max_pages=512, **kw), code, "workspace")


def test_followed_weights_past_a_grid_are_refused(lib):
    """B * H workgroups of 256 threads join pieces and B * Hk or more add weights, in one launch: 2^32
    threads do not start."""
    def call(B, H, pages, **kw):
        c = struct(D=64, Hk=1, **kw)
        return lib.ugbsa_paged_decode_mass(ctypes.addressof(c), 16, 64, 64, 64, 1, H, 16, 16, 8, B, pages, 0.1, None, None, 0,
                                           16, 4096, 4096, 16, 64, 64, 1, 16, 0, None)
    refused(lib, call(65535, 256, 17), -1, "too large")          # 16776960 + 65535 workgroups
    refused(lib, call(65535, 255, 17), -1, "workspace")          # 16711425 + 65535: as far as the next check
    refused(lib, call(65535, 256, 16), -1, "workspace")          # rows of one workgroup: the grids have two dimensions


def test_evictions_past_a_grid_are_refused(lib):
    """A workgroup of up to 1024 threads a row, and one of 256 a new page: 2^32 threads or more do not start."""
    def evict(Hk=2, B=1, new_pages=4):
        c = four(Hk=Hk)
        return lib.ugbsa_paged_evict(ctypes.addressof(c), 16, 0, 0, 16, 16, 8, B, 8, 16, 4, new_pages, 100, 0, 0, 16, 16,
                                     16, 256, 256, None, 0, None)
    refused(lib, evict(new_pages=1 << 24), -1, "new_pages")
    refused(lib, evict(Hk=65, B=65535), -1, "2^22")
    refused(lib, evict(Hk=65535, B=65535), -1, "2^22")


def test_write_rotary_refusals(lib):
    c = four()

    def write(turns=16, r=64, attention=1.0, positions=16, T=4, k=16, cache=c, table=True):
        t = _capi.RotaryStruct(turns=turns, rotary_dim=r, interleaved=0, attention=attention)
        return lib.ugbsa_paged_write_rotary(ctypes.addressof(cache) if cache else None, k, 256, 128, 1, 16, 256, 128, 1,
                                            16, 16, 16, 8, 1, T, 8, ctypes.addressof(t) if table else None, positions, None)
    refused(lib, write(cache=None), -1, "cache is null")
    refused(lib, write(table=False), -1, "table")
    refused(lib, write(turns=None), -1, "table")
    refused(lib, write(r=130), -1, "rotary_dim")
    refused(lib, write(attention=float("inf")), -1, "attention")
    refused(lib, write(positions=2), -2, "positions")
    refused(lib, write(k=None), -1, "k is null")
    assert write(T=0) == 0


@pytest.mark.filterwarnings("ignore")
def test_weights_with_tangents_or_gradients_are_refused(monkeypatch):
    monkeypatch.setattr(pc, "_launch", lambda *a: None)
    cache, q = host_cache(), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    table, lens, new = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.ones(1, 2, dtype=torch.int32)
    mass = torch.zeros(1, 2, 128)
    seen = mass._version
    pc.paged_decode(q, cache, table, lens, 0.1, mass=mass)
    assert mass._version > seen                             # autograd sees the change
    pc.paged_evict(cache, mass, table, lens, new, 64)
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        dual = fw.make_dual(mass, torch.ones_like(mass))
        for call in (lambda: pc.paged_decode(q, cache, table, lens, 0.1, mass=dual),
                     lambda: pc.paged_evict(cache, dual, table, lens, new, 64)):
            with pytest.raises(AssertionError, match="forward-mode"):
                call()
    for bad in (mass.clone().requires_grad_(), torch._neg_view(mass.clone()), mass.double(), mass[..., :64]):
        for call in (lambda: pc.paged_decode(q, cache, table, lens, 0.1, mass=bad),
                     lambda: pc.paged_evict(cache, bad, table, lens, new, 64)):
            with pytest.raises(AssertionError, match="mass"):
                call()


def test_keys_are_turned_by_whole_arguments_only(monkeypatch):
    monkeypatch.setattr(pc, "_launch", lambda *a: None)
    from types import SimpleNamespace
    cache, k = host_cache(), torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    rot = SimpleNamespace(_call=(None, -1, 64))
    pc.paged_write(cache, k, k, table, lens, rotary=rot)
    pc.paged_write(cache, k, k, table, lens, rotary=rot, positions=lens)
    for kw in (dict(positions=lens), dict(rotary=SimpleNamespace(_call=(None, -1, 128))),
               dict(rotary=SimpleNamespace(_call=(None, 0, 64))), dict(rotary=rot, positions=lens.long()),
               dict(rotary=rot, positions=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(AssertionError):
            pc.paged_write(cache, k, k, table, lens, **kw)


def test_tensors_made_for_inference(monkeypatch):
    """They keep no version that a call in place could raise."""
    import rotary as ro
    from types import SimpleNamespace
    monkeypatch.setattr(pc, "_launch", lambda *a: None)
    monkeypatch.setattr(ro, "_launch", lambda *a: None)
    with torch.inference_mode():
        cache, q = host_cache(), torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
        table, lens, mass = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, 128)
        pc.paged_decode(q, cache, table, lens, 0.1, mass=mass)
        pc.paged_evict(cache, mass, table, lens, torch.ones(1, 2, dtype=torch.int32), 64)
        x = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
        ro.rotary(SimpleNamespace(_call=(None, -1, 64)), lens, x, out=x)
    pc.paged_decode(q, cache, table, lens, 0.1, mass=mass)
