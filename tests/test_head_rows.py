"""Norms with the position rotation and 8-bit caches on the CPU: the calls that are refused,
and their oracle."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import head_rows as hr
from varlenabsorbflashattn_amd import (_lib, packed_qk_norm_rope, paged_chunk_attn,
                                       paged_decode_attn, paged_kv_append, paged_kv_gather)

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _rows(dt=torch.bfloat16, T=3, H=4, Hk=2, D=64):
    return {"q": torch.zeros(T, H, D, dtype=dt), "k": torch.zeros(T, Hk, D, dtype=dt),
            "positions": torch.zeros(T, dtype=torch.int32), "inv_freq": torch.zeros(D // 2),
            "q_weight": torch.ones(D), "k_weight": torch.ones(D)}


REFUSED_ROWS = [
    ({"q": torch.zeros(3, 64, dtype=torch.bfloat16)}, ValueError, "expected 3-D"),
    ({"q": torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)}, ValueError, "batch=1"),
    ({"k": torch.zeros(2, 2, 64, dtype=torch.bfloat16)}, AssertionError, "q and k must be"),
    ({"k": torch.zeros(3, 2, 32, dtype=torch.bfloat16)}, AssertionError, "q and k must be"),
    ({"k": torch.zeros(3, 2, 64, dtype=torch.float16)}, AssertionError, "share dtype"),
    ({"positions": None}, AssertionError, "needs positions"),
    ({"positions": torch.zeros(2, dtype=torch.int32)}, AssertionError, "positions must be"),
    ({"positions": torch.zeros(3, dtype=torch.int64)}, AssertionError, "int32"),
    ({"positions": torch.zeros(1, dtype=torch.int32).expand(3)}, ValueError, "contiguous"),
    ({"inv_freq": torch.zeros(33)}, AssertionError, "inv_freq must be"),
    ({"inv_freq": torch.zeros(32, dtype=torch.float64)}, AssertionError, "float32"),
    ({"inv_freq": torch.zeros(1).expand(32)}, ValueError, "contiguous"),
    ({"inv_freq": torch.zeros(32, requires_grad=True)}, ValueError, "no gradient"),
    ({"inv_freq": None, "rot_scale": 2.0}, ValueError, "rot_scale belongs"),
    ({"q_weight": torch.ones(32)}, AssertionError, r"must be \[D\]"),
    ({"q_weight": torch.ones(64, dtype=torch.float16)}, AssertionError, "float32 or of"),
    ({"q_weight": torch.ones(64, dtype=torch.bfloat16)}, AssertionError, "share dtype"),
    ({"k_weight": torch.ones(1).expand(64)}, ValueError, "contiguous"),
    ({}, AssertionError, "requires GPU tensors"),
]


@pytest.mark.parametrize("change,error,text", REFUSED_ROWS)
def test_refused_rows(change, error, text):
    a = _rows()
    a.update(change)
    with pytest.raises(error, match=text):
        packed_qk_norm_rope(a.pop("q"), a.pop("k"), **a)


def test_refused_row_types_and_tangents():
    a = _rows(torch.float32)
    with pytest.raises(AssertionError, match="dtype not supported"):
        packed_qk_norm_rope(a.pop("q"), a.pop("k"), **a)
    import torch.autograd.forward_ad as fwAD
    a = _rows()
    with fwAD.dual_level():
        q = fwAD.make_dual(a.pop("q"), torch.ones(3, 4, 64, dtype=torch.bfloat16))
        with pytest.raises(ValueError, match="forward-mode"):
            packed_qk_norm_rope(q, a.pop("k"), **a)


def _cache(dt=torch.bfloat16, n=3, T=3, H=4, Hk=2, D=64, pages=5, page=16, width=2):
    return {"k": torch.zeros(T, Hk, D, dtype=dt), "v": torch.zeros(T, Hk, D, dtype=dt),
            "q": torch.zeros(T, H, D, dtype=dt),
            "k_cache": torch.zeros(pages, page, Hk, D).to(E4M3),
            "v_cache": torch.zeros(pages, page, Hk, D).to(E4M3),
            "page_table": torch.zeros(n, width, dtype=torch.int32),
            "cache_lens": torch.zeros(n, dtype=torch.int32),
            "k_scale": torch.full((pages, page, Hk), 127, dtype=torch.uint8).view(E8M0),
            "v_scale": torch.full((pages, page, Hk), 127, dtype=torch.uint8).view(E8M0)}


def _append(a):
    a = dict(a)
    pos = [a.pop(x) for x in ("k", "v", "k_cache", "v_cache", "page_table", "cache_lens")]
    return paged_kv_append(*pos, **a)


def _gather(a):
    kw = {x: a[x] for x in ("k_scale", "v_scale") if x in a}
    return paged_kv_gather(a["k_cache"], a["v_cache"], a["page_table"],
                           torch.zeros(len(a["page_table"]) + 1, dtype=torch.int32), 4,
                           dtype=a["k"].dtype, **kw)


def _decode(a):
    return paged_decode_attn(a["q"], a["k_cache"], a["v_cache"], a["page_table"], a["cache_lens"],
                             k_scale=a["k_scale"], v_scale=a["v_scale"])


def _chunk(a, cu=torch.zeros(4, dtype=torch.int32), **kw):
    return paged_chunk_attn(a["q"], a["k_cache"], a["v_cache"], a["page_table"], a["cache_lens"],
                            cu, k_scale=a["k_scale"], v_scale=a["v_scale"], **kw)


REFUSED_CODES = [
    ({"k_scale": None, "v_scale": None}, AssertionError, "need k_scale and v_scale"),
    ({"v_scale": None}, AssertionError, "belong together"),
    ({"k_cache": torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)}, AssertionError,
     "must be float8_e4m3fn"),
    ({"v_cache": torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)}, AssertionError, "share dtype"),
    ({"k_scale": torch.zeros(5, 16, 2)}, AssertionError, "float8_e8m0fnu"),
    ({"v_scale": torch.zeros(5, 16, 1, dtype=torch.uint8).view(E8M0)}, AssertionError,
     r"must be \[n_pages"),
    ({"k_scale": torch.zeros(5, 16, 1, dtype=torch.uint8).view(E8M0).expand(5, 16, 2)}, ValueError,
     "expanded"),
    ({"k_cache": torch.zeros(5, 16, 2, 72).to(E4M3)[..., :64]}, ValueError, "multiples of 16"),
    ({}, AssertionError, "requires GPU tensors"),
]


@pytest.mark.parametrize("call", [_append, _gather, _decode, _chunk])
@pytest.mark.parametrize("change,error,text", REFUSED_CODES)
def test_refused_codes(call, change, error, text):
    a = _cache()
    a.update(change)
    with pytest.raises(error, match=text):
        call(a)


def test_refused_append_options():
    def refused(error, text, **kw):
        a = _cache()
        a.update(kw)
        with pytest.raises(error, match=text):
            _append(a)
    refused(AssertionError, "dtype and device", q=torch.zeros(3, 4, 64, dtype=torch.float16))
    refused(AssertionError, "q_weight needs q", q=None, q_weight=torch.ones(64))
    refused(AssertionError, r"must be \[D\]", k_weight=torch.ones(63))
    refused(ValueError, "rot_scale belongs", rot_scale=0.5)
    refused(ValueError, "no backward", k_weight=torch.ones(64, requires_grad=True))
    a = _cache(torch.float32)
    with pytest.raises(AssertionError, match="dtype not supported"):
        _append(a)


def test_refused_gather_options():
    a = _cache()
    cu = torch.zeros(4, dtype=torch.int32)

    def refused(error, text, cu=cu, total=4, dtype=torch.bfloat16, starts=None, cache=a["k_cache"],
                scales=True):
        kw = {"k_scale": a["k_scale"], "v_scale": a["v_scale"]} if scales else {}
        with pytest.raises(error, match=text):
            paged_kv_gather(cache, cache, a["page_table"], cu, total, starts=starts, dtype=dtype,
                            **kw)
    refused(ValueError, "total", total=-1)
    refused(AssertionError, "cu_seqlens", cu=cu[:3])
    refused(AssertionError, "int32", cu=cu.long())
    refused(AssertionError, "starts must be", starts=cu)
    refused(AssertionError, "int32", starts=cu[:3].long())
    refused(AssertionError, "need the dtype", dtype=None)
    refused(AssertionError, "not supported", dtype=torch.float32)
    half = torch.zeros(5, 16, 2, 64, dtype=torch.float16)
    refused(AssertionError, "comes back in its dtype", cache=half, scales=False)


def test_refused_chunk_options():
    def refused(error, text, cu=torch.zeros(4, dtype=torch.int32), change={}, **kw):
        a = _cache()
        a.update(change)
        with pytest.raises(error, match=text):
            _chunk(a, cu, **kw)
    refused(AssertionError, "cu_seqlens must be", cu=torch.zeros(3, dtype=torch.int32))
    refused(AssertionError, "int32", cu=torch.zeros(4, dtype=torch.int64))
    refused(ValueError, "contiguous", cu=torch.zeros(1, dtype=torch.int32).expand(4))
    for cap in (0.0, -1.0, float("nan"), 1e-50):
        refused(ValueError, "softcap must be positive", softcap=cap)
    refused(ValueError, "window must be positive", window=0)
    refused(AssertionError, r"alibi_slopes must be \[H\]", alibi_slopes=torch.zeros(3))
    refused(AssertionError, "q must be", change={"q": torch.zeros(3, 4, 32, dtype=torch.bfloat16)})
    refused(AssertionError, "not supported", change={"q": torch.zeros(3, 4, 64)})
    refused(ValueError, "no backward",
            change={"q": torch.zeros(3, 4, 64, dtype=torch.bfloat16, requires_grad=True)})


def test_refused_by_the_c_abi():
    """What the entry points themselves refuse, before any launch (no GPU needed)."""
    L = _lib.lib()
    x = 1 << 24
    BF = _lib.DT_BF16

    def cache(**kw):
        c = _lib.PagedCache(k=1 << 20, v=1 << 21, n_pages=5, page_size=16, Hk=2, D=64,
                            k_page=2048, k_token=128, k_head=64, v_page=2048, v_token=128,
                            v_head=64, page_table=1 << 22, table_stride=2, table_width=2,
                            cache_lens=1 << 23, n_seq=3)
        for n, v in kw.items():
            setattr(c, n, v)
        return C.byref(c)

    def scales(**kw):
        s = _lib.RowScales(k=1 << 20, v=1 << 21, k_page=32, k_token=2, k_head=1, v_page=32,
                           v_token=2, v_head=1)
        for n, v in kw.items():
            setattr(s, n, v)
        return C.byref(s)

    def all_refused(call, args, bad, rc=_lib.VAFA_ERR_VALUE):
        for at, value in bad:
            a = [value if i == at else y for i, y in enumerate(args)]
            assert call(*a) == rc, (at, value)

    store = [cache(), scales(), x, 128, 64, x, 128, 64, 3, None, x, 256, 64, 4, x, x, 64, 0, 1.0, x,
             x, 1, 1e-6, BF, None]
    all_refused(L.vafa_paged_store, store, [
        (0, cache(k_token=136)), (0, cache(v=8)), (1, scales(k=None)), (1, scales(v_token=-1)),
        (2, x + 8), (3, 4), (8, 4), (8, -1), (10, x + 2), (13, -1), (14, None), (15, None),
        (16, 8), (16, 80), (16, -16), (18, float("inf")), (22, -1.0), (22, float("nan"))])
    all_refused(L.vafa_paged_store, store, [(0, cache(D=96)), (23, _lib.DT_F32)],
                _lib.VAFA_ERR_ASSERT)
    gather = [cache(), scales(), x, x, 7, x, x, BF, None]
    all_refused(L.vafa_paged_gather, gather, [
        (0, cache(n_pages=0)), (0, cache(k_page=24)), (1, scales(v=None)), (2, None), (4, -1),
        (4, 1 << 40), (5, None), (6, x + 8), (0, cache(page_table=None))])
    all_refused(L.vafa_paged_gather, gather, [(0, cache(D=24)), (7, 0)], _lib.VAFA_ERR_ASSERT)
    fwd = [x, 256, 64, 4, x, 128, 64, 2, 7, 64, x, x, 64, 0, 1.0, x, x, 1, 1e-6, x, x, BF, None]
    all_refused(L.vafa_qk_norm_rope_fwd, fwd, [
        (0, x + 4), (1, 12), (3, 0), (3, 1 << 20), (4, None), (6, -8), (7, 0), (8, -1), (8, 1 << 31),
        (10, None), (11, None), (12, 24), (14, float("nan")), (18, float("inf")), (19, None),
        (20, x + 8)])
    all_refused(L.vafa_qk_norm_rope_fwd, fwd, [(9, 80), (21, 7)], _lib.VAFA_ERR_ASSERT)
    need = L.vafa_qk_norm_rope_bwd_workspace(7, 4, 2, 64)
    assert need > 0 and L.vafa_qk_norm_rope_bwd_workspace(7, 0, 2, 64) == -1
    bwd = fwd[:19] + [x, x, x, x, x, x, BF, x, need, None]
    all_refused(L.vafa_qk_norm_rope_bwd, bwd, [
        (0, None), (15, None), (16, None), (19, None), (20, x + 8), (21, None), (22, x + 2)])
    all_refused(L.vafa_qk_norm_rope_bwd, bwd, [(26, None), (27, need - 1)],
                _lib.VAFA_ERR_WORKSPACE)
    wide = cache(table_width=100)
    need = L.vafa_paged_chunk_workspace(wide, 7, 4, 0)
    assert need > 0 and L.vafa_paged_chunk_workspace(cache(), 7, 4, 0) == 0
    for c, T, H, window in ((cache(n_pages=0), 7, 4, 0), (cache(D=96), 7, 4, 0), (wide, -1, 4, 0),
                            (wide, 1 << 31, 4, 0), (wide, 7, 3, 0), (wide, 7, 8192, 0),
                            (wide, 7, 4, -1)):
        assert L.vafa_paged_chunk_workspace(c, T, H, window) == -1
    chunk = [wide, scales(), x, 256, 64, 7, 4, x, x, 0.125, 0.0, 0, None, BF, x, need, None]
    all_refused(L.vafa_paged_chunk, chunk, [
        (0, cache(k_token=136, table_width=100)), (1, scales(k=None)), (2, x + 2), (3, 12), (7, None),
        (8, None), (9, float("nan")), (10, -1.0), (10, 1e-40), (11, -1)])
    all_refused(L.vafa_paged_chunk, chunk, [(13, 0), (6, 5)], _lib.VAFA_ERR_ASSERT)
    all_refused(L.vafa_paged_chunk, chunk, [(14, None), (14, x + 8), (15, need - 1)],
                _lib.VAFA_ERR_WORKSPACE)
    # no rows: nothing is launched
    assert L.vafa_paged_chunk(*[0 if i == 5 else y for i, y in enumerate(chunk)]) == 0
    assert L.vafa_qk_norm_rope_fwd(*[0 if i == 8 else y for i, y in enumerate(fwd)]) == 0
    assert L.vafa_paged_gather(*[0 if i == 4 else y for i, y in enumerate(gather)]) == 0


def test_oracle_codes_are_e4m3():
    """The oracle's rounding against torch's own conversion, and its exponents by their
    definition."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((500, 64)) * 2.0 ** rng.integers(-30, 30, (500, 1))
    x[0], x[1, 1:], x[2] = 0.0, 0.0, np.ldexp(448.0, -3)
    x = x.astype(np.float32).astype(np.float64)
    e = hr.row_exponents(x, "bf16")
    amax = np.abs(x).max(1)
    some = amax > 0
    assert (amax <= np.ldexp(448.0, e))[some].all() and (amax > np.ldexp(448.0, e - 1))[some].all()
    assert e[0] == 0 and e[2] == -3
    got = hr.to_code(x, e[:, None], "bf16")
    want = torch.from_numpy(np.ldexp(x, -e[:, None]).astype(np.float32)).to(E4M3).double().numpy()
    assert np.array_equal(got, np.ldexp(want, e[:, None]))


def test_oracle_limits_of_the_types():
    """Codes of the largest numbers of a type stand for numbers that it holds."""
    for kind, dt in (("bf16", torch.bfloat16), ("fp16", torch.float16)):
        big = torch.finfo(dt).max
        x = np.array([[big, -big, big / 3, 1.0, 0.0, np.inf, np.nan, big * 0.9]])
        e = hr.row_exponents(x, kind)
        assert e[0] == hr.TOP[kind]
        y = hr.to_code(x, e[:, None], kind)
        assert np.isfinite(torch.from_numpy(y[:, :5]).to(dt).float().numpy()).all()
        assert np.isnan(y[0, 5:7]).all()
        assert y[0, 0] == np.ldexp(240.0, hr.TOP[kind])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rot", [0, 16, 32])
def test_oracle_gradients(rot, inter):
    """The oracle's backward against differences of its forward."""
    rng = np.random.default_rng(rot + inter)
    x, dy = rng.standard_normal((2, 3, 2, 32))
    w, pos = 1 + 0.2 * rng.standard_normal(32), np.array([0, 5, 1000])
    inv = 10000.0 ** (-np.arange(0, rot, 2) / max(rot, 1)) if rot else None
    args = (pos, inv, inter)

    def loss(x, w):
        return (hr.forward(x, *args, w, 1e-3, 1.3)[0] * dy).sum()
    dx, mag, dw, wmag = hr.backward(x, dy, *args, w, 1e-3, 1.3)
    h = 1e-5
    for _ in range(20):
        i = tuple(rng.integers(0, n) for n in x.shape)
        d = np.zeros_like(x)
        d[i] = h
        assert math.isclose((loss(x + d, w) - loss(x - d, w)) / (2 * h), dx[i], rel_tol=1e-6,
                            abs_tol=1e-7)
        d = np.zeros_like(w)
        d[i[2]] = h
        assert math.isclose((loss(x, w + d) - loss(x, w - d)) / (2 * h), dw[i[2]], rel_tol=1e-6,
                            abs_tol=1e-7)
    assert (np.abs(dx) <= mag + 1e-12).all() and (np.abs(dw) <= wmag + 1e-12).all()


def test_row_strides_of_the_c_abi():
    """Strides past 32 bits: refused by the entry points whose kernels take 32-bit factors, as
    before no error of the others (no rows: nothing is launched)."""
    L, x, far, BF = _lib.lib(), 1 << 24, 1 << 33, _lib.DT_BF16
    c = _lib.PagedCache(k=1 << 20, v=1 << 21, n_pages=5, page_size=16, Hk=2, D=64, k_page=2048,
                        k_token=128, k_head=64, v_page=2048, v_token=128, v_head=64,
                        page_table=1 << 22, table_stride=2, table_width=2, cache_lens=1 << 23,
                        n_seq=0)
    c = C.byref(c)
    append = [c, x, far, 64, x, far, far, 0, None, x, far, far, 4, x, x, 64, 0, BF, None]
    assert L.vafa_paged_append(*append) == 0
    decode = [c, x, far, far, 4, x, 0.125, 0.0, 0, None, BF, x, 1 << 20, None]
    assert L.vafa_paged_decode(*decode) == 0
    store = [c, None, x, 128, 64, x, 128, 64, 0, None, x, 256, 64, 4, x, x, 64, 0, 1.0, x, x, 1,
             1e-6, BF, None]
    assert L.vafa_paged_store(*store) == 0
    for at in (3, 4, 6, 7, 11, 12):
        assert L.vafa_paged_store(*[far if i == at else y for i, y in enumerate(store)]) == \
            _lib.VAFA_ERR_VALUE, at


def test_gather_names_its_argument():
    """cu_seqlens stands in for lengths inside: errors name it all the same."""
    kc, table = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="cu_seqlens must be int32"):
        paged_kv_gather(kc, kc, table, torch.tensor([0, 1, 2]), 2)
    with pytest.raises(ValueError, match="cu_seqlens must be contiguous"):
        paged_kv_gather(kc, kc, table, torch.zeros(6, dtype=torch.int32)[::2], 2)


def test_refused_types_name_whose_they_differ_from():
    """A cache of codes is float8: rows that go into it have to be of k's dtype, not the cache's."""
    for name in ("q", "v"):
        a = _cache()
        a[name] = a[name].to(torch.float16)
        with pytest.raises(AssertionError, match=f"{name} must have k's dtype and device"):
            _append(a)
        for x in ("k_cache", "v_cache"):
            a[x] = torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)
        a["k_scale"] = a["v_scale"] = None
        with pytest.raises(AssertionError, match=f"{name} must have the cache's dtype and device"):
            _append(a)


def test_far_strides_of_chunks():
    """Strides of pages and tokens reach 2^35 elements in 16 bits and 2^36 codes, which are as many
    pieces of 16 bytes (no rows: nothing is launched)."""
    L, x = _lib.lib(), 1 << 24

    def rc(codes, **far):
        c = _lib.PagedCache(k=1 << 20, v=1 << 21, n_pages=5, page_size=16, Hk=2, D=64, k_page=2048,
                            k_token=128, k_head=64, v_page=2048, v_token=128, v_head=64,
                            page_table=1 << 22, table_stride=2, table_width=2,
                            cache_lens=1 << 23, n_seq=3)
        for n, v in far.items():
            setattr(c, n, v)
        s = _lib.RowScales(k=1 << 20, v=1 << 21, k_page=32, k_token=2, k_head=1, v_page=32,
                           v_token=2, v_head=1)
        return L.vafa_paged_chunk(C.byref(c), C.byref(s) if codes else None, x, 256, 64, 0, 4, x, x,
                                  0.125, 0.0, 0, None, _lib.DT_BF16, None, 0, None)
    for name in ("k_page", "k_token", "v_page", "v_token"):
        for codes, limit in ((False, 1 << 35), (True, 1 << 36)):
            assert rc(codes, **{name: limit - 16}) == 0, (name, codes)
            assert rc(codes, **{name: limit}) == _lib.VAFA_ERR_VALUE, (name, codes)
