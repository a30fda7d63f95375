"""The paged-cache operators on the CPU: page lookups and the decoding attention's split
under host sanitizers, the calls that are refused, and their oracle."""
import os
import shutil
import subprocess
import tempfile

import numpy as np
import pytest
import torch

from conftest import ROOT
from oracle import paged as op
from varlenabsorbflashattn_amd import _lib, paged_decode_attn, paged_kv_append


def test_paged_addressing_under_host_sanitizers():
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    tmp = tempfile.mkdtemp()
    try:
        exe = os.path.join(tmp, "paged_fuzz")
        subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-Wno-unknown-pragmas",
                        "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                        "-I", os.path.join(ROOT, "varlenabsorbflashattn_amd", "csrc"),
                        os.path.join(ROOT, "tests", "host_fuzz", "paged_fuzz.cpp"), "-o", exe],
                       check=True, capture_output=True, text=True)
        for seed in (3, 99):
            r = subprocess.run([exe, "400", str(seed)], capture_output=True, text=True, timeout=300)
            assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
            assert "0 failed checks" in r.stdout
    finally:
        shutil.rmtree(tmp, ignore_errors=True)


def _args(dt=torch.bfloat16, n=3, T=3, H=4, Hk=2, D=64, pages=5, page=16, width=2):
    return {"q": torch.zeros(T, H, D, dtype=dt), "k": torch.zeros(T, Hk, D, dtype=dt),
            "v": torch.zeros(T, Hk, D, dtype=dt),
            "k_cache": torch.zeros(pages, page, Hk, D, dtype=dt),
            "v_cache": torch.zeros(pages, page, Hk, D, dtype=dt),
            "page_table": torch.zeros(n, width, dtype=torch.int32),
            "cache_lens": torch.zeros(n, dtype=torch.int32)}


def _append(a, **kw):
    pos = [a[x] for x in ("k", "v", "k_cache", "v_cache", "page_table", "cache_lens")]
    return paged_kv_append(*pos, q=a["q"], **kw)


def _decode(a, **kw):
    pos = [a[x] for x in ("q", "k_cache", "v_cache", "page_table", "cache_lens")]
    return paged_decode_attn(*pos, **kw)


REFUSED = [
    # (what is changed, to what, error, part of its text)
    ("k_cache", torch.zeros(5, 16, 64, dtype=torch.bfloat16), AssertionError, "n_pages, page_size"),
    ("v_cache", torch.zeros(5, 8, 2, 64, dtype=torch.bfloat16), AssertionError, "alike"),
    ("v_cache", torch.zeros(5, 16, 2, 64, dtype=torch.float16), AssertionError, "share dtype"),
    ("page_table", torch.zeros(3, dtype=torch.int32), AssertionError, "page_table must be"),
    ("page_table", torch.zeros(2, 2, dtype=torch.int32), AssertionError, "page_table must be"),
    ("page_table", torch.zeros(3, 2, dtype=torch.int64), AssertionError, "must be int32"),
    ("cache_lens", torch.zeros(3, dtype=torch.int64), AssertionError, "must be int32"),
    ("cache_lens", torch.zeros(3, 1, dtype=torch.int32), AssertionError, "cache_lens"),
]


@pytest.mark.parametrize("call", [_append, _decode])
@pytest.mark.parametrize("name,value,error,text", REFUSED)
def test_refused_caches(call, name, value, error, text):
    a = _args()
    a[name] = value
    with pytest.raises(error, match=text):
        call(a)


@pytest.mark.parametrize("call", [_append, _decode])
def test_refused_types_and_devices(call):
    with pytest.raises(AssertionError, match="dtype not supported"):
        call(_args(torch.float32))
    with pytest.raises(AssertionError, match="requires GPU tensors"):
        call(_args())
    for name in ("q", "k_cache"):
        a = _args()
        a[name].requires_grad_(True)
        with pytest.raises(ValueError, match="no backward"):
            call(a)
        with torch.no_grad(), pytest.raises(AssertionError, match="requires GPU"):
            call(a)


def test_refused_decode_options():
    for kw in ({"softcap": 0.0}, {"softcap": -1.0}, {"softcap": float("nan")}, {"softcap": 1e-50}):
        with pytest.raises(ValueError, match="softcap must be positive"):
            _decode(_args(), **kw)
    for w in (0, -3):
        with pytest.raises(ValueError, match="window must be positive"):
            _decode(_args(), window=w)


def test_refused_by_the_c_abi():
    """What the entry points themselves refuse, before any launch (no GPU needed)."""
    import ctypes as C
    L = _lib.lib()

    def cache(**kw):
        c = _lib.PagedCache(k=1 << 20, v=1 << 21, n_pages=5, page_size=16, Hk=2, D=64,
                            k_page=2048, k_token=128, k_head=64, v_page=2048, v_token=128,
                            v_head=64, page_table=1 << 22, table_stride=2, table_width=2,
                            cache_lens=1 << 23, n_seq=3)
        for n, v in kw.items():
            setattr(c, n, v)
        return C.byref(c)

    for c in (cache(n_pages=0), cache(page_size=0), cache(Hk=0), cache(k_token=12), cache(v=4),
              cache(n_seq=-1), cache(table_width=-1)):
        assert L.vafa_paged_decode_workspace(c, 4, 0) == -1
    for H, window, kw in ((3, 0, {}), (0, 0, {}), (4, -1, {}), (4, 0, {"D": 96}),
                          (4, 0, {"table_width": (1 << 31) - 1, "page_size": 1 << 20,
                                  "n_seq": 4096})):
        assert L.vafa_paged_decode_workspace(cache(**kw), H, window) == -1
    # short sequences need no partial results
    assert L.vafa_paged_decode_workspace(cache(), 4, 0) == 0
    need = L.vafa_paged_decode_workspace(cache(table_width=100), 4, 0)
    assert need > 0
    x = 1 << 24
    dec = [cache(table_width=100), x, 256, 64, 4, x, 0.125, 0.0, 0, None, _lib.DT_BF16, x, need, None]

    def rc(at, value, call=L.vafa_paged_decode, args=dec):
        return call(*[value if i == at else y for i, y in enumerate(args)])

    assert rc(12, need - 1) == _lib.VAFA_ERR_WORKSPACE
    assert rc(11, None) == _lib.VAFA_ERR_WORKSPACE
    assert rc(10, _lib.DT_F32) == _lib.VAFA_ERR_ASSERT
    for at, bad in ((1, x + 2), (2, 100), (6, float("nan")), (7, -1.0), (7, float("inf")), (7, 1e-40),
                    (7, 2e4), (6, 3e38), (8, -1)):
        assert rc(at, bad) == _lib.VAFA_ERR_VALUE, at
    app = [cache(), x, 128, 64, x, 128, 64, 3, None, x, 256, 64, 4, x, x, 64, 0, _lib.DT_BF16, None]
    for at, bad in ((1, x + 8), (2, 4), (5, -8), (7, 4), (7, -1), (9, x + 2), (12, -1), (15, 63),
                    (15, 66), (15, -2)):
        assert rc(at, bad, L.vafa_paged_append, app) == _lib.VAFA_ERR_VALUE, at
    assert rc(0, cache(D=60), L.vafa_paged_append, app) == _lib.VAFA_ERR_ASSERT
    assert "head_dim 60" in _lib.last_error()
    # more blocks of 256 threads than a launch can have
    big = list(app)
    big[0], big[7], big[8] = cache(n_seq=1 << 20), (1 << 31) - 1, x
    assert L.vafa_paged_append(*big) == _lib.VAFA_ERR_VALUE and "too many" in _lib.last_error()
    assert rc(0, cache(n_seq=1 << 18, table_width=1), L.vafa_paged_decode,
              dec[:4] + [128] + dec[5:]) == _lib.VAFA_ERR_VALUE
    # nothing to do: no launch
    app[7], app[8] = 0, x
    assert L.vafa_paged_append(*app) == _lib.VAFA_OK
    assert rc(0, cache(n_seq=0)) == _lib.VAFA_OK


def test_oracle_decode_against_softmax():
    g = np.random.default_rng(0)
    q = g.standard_normal((1, 2, 8))
    k, v = g.standard_normal((2, 4, 3, 1, 8))
    table = np.array([[2, 0, 3]], np.int32)
    out, mag, flat = op.decode(q, k, v, table, [7], 0.5)
    rows = np.concatenate([k[2], k[0], k[3]])[:7, 0], np.concatenate([v[2], v[0], v[3]])[:7, 0]
    P = torch.softmax(torch.from_numpy(0.5 * q[0] @ rows[0].T), 1).numpy()
    np.testing.assert_allclose(out[0], P @ rows[1], rtol=1e-12)
    assert (mag >= np.abs(out) - 1e-12).all()
    # a page outside the cache and a length past the table
    table[0, 1] = 9
    out, _, _ = op.decode(q, k, v, table, [100], 0.5)
    keep = np.concatenate([k[2], k[3]])[:, 0], np.concatenate([v[2], v[3]])[:, 0]
    P = torch.softmax(torch.from_numpy(0.5 * q[0] @ keep[0].T), 1).numpy()
    np.testing.assert_allclose(out[0], P @ keep[1], rtol=1e-12)


@pytest.mark.parametrize("call", [_append, _decode])
@pytest.mark.parametrize("name,shape", [("page_table", (3, 2)), ("cache_lens", (3,))])
def test_expanded_index_tensors_are_refused(call, name, shape):
    """One element stands for a row: the kernels would read behind it."""
    a = _args()
    a[name] = torch.zeros(1, dtype=torch.int32).expand(shape)
    with pytest.raises(ValueError, match="must be contiguous"):
        call(a)
    # rows that all sequences share are whole rows
    a["page_table"], a["cache_lens"] = torch.zeros(1, 2, dtype=torch.int32).expand(3, 2), \
        torch.zeros(3, dtype=torch.int32)
    with pytest.raises(AssertionError, match="requires GPU tensors"):
        call(a)


def test_expanded_vectors_are_refused():
    one = torch.ones(1)
    for kw, text in (({"cu_seqlens": torch.zeros(1, dtype=torch.int32).expand(4)}, "cu_seqlens"),
                     ({"inv_freq": one.expand(32)}, "inv_freq")):
        with pytest.raises(ValueError, match=text + " must be contiguous"):
            _append(_args(), **kw)
    with pytest.raises(ValueError, match="alibi_slopes must be contiguous"):
        _decode(_args(), alibi_slopes=one.expand(4))
    # one head, one frequency: any stride
    for call, kw in ((_append, {"inv_freq": torch.ones(4)[::4]}),
                     (_decode, {"alibi_slopes": torch.ones(4)[::4]})):
        with pytest.raises(AssertionError, match="requires GPU tensors"):
            call(_args(H=1, Hk=1), **kw)


@pytest.mark.parametrize("call,names", [(_append, ("q", "k", "v", "k_cache", "v_cache")),
                                        (_decode, ("q", "k_cache", "v_cache"))])
def test_tangents_and_traces_are_refused(call, names):
    import torch.autograd.forward_ad as fw
    for name in names:
        a = _args()
        with fw.dual_level(), torch.no_grad():
            a[name] = fw.make_dual(a[name], torch.ones_like(a[name]))
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                call(a)
    a = _args()
    with pytest.raises(ValueError, match="cannot be traced"):
        torch.jit.trace(lambda q: call({**a, "q": q}), (a["q"],))


def test_missing_pointers_are_refused_by_the_c_abi():
    """NULL where there is something to read or write is an error, not an access."""
    import ctypes as C
    L = _lib.lib()

    def cache(**kw):
        c = {"k": 1 << 20, "v": 1 << 21, "n_pages": 5, "page_size": 16, "Hk": 2, "D": 64,
             "k_page": 2048, "k_token": 128, "k_head": 64, "v_page": 2048, "v_token": 128,
             "v_head": 64, "page_table": 1 << 22, "table_stride": 2, "table_width": 2,
             "cache_lens": 1 << 23, "n_seq": 3, **kw}
        return C.byref(_lib.PagedCache(**c))
    x = 1 << 24
    dec = [cache(), x, 256, 64, 4, x, 0.125, 0.0, 0, None, _lib.DT_BF16, None, 0, None]
    app = [cache(), x, 128, 64, x, 128, 64, 3, None, x, 256, 64, 4, x, x, 64, 0, _lib.DT_BF16, None]
    for call, args, at in ((L.vafa_paged_decode, dec, (1, 5)),
                           (L.vafa_paged_append, app, (1, 4, 9, 13, 14))):
        bad = [(i, None) for i in at] + [(0, cache(**{n: None})) for n in
                                         ("k", "v", "page_table", "cache_lens")]
        for i, value in bad:
            rc = call(*[value if j == i else y for j, y in enumerate(args)])
            assert rc == _lib.VAFA_ERR_VALUE and "NULL" in _lib.last_error(), (call, i)
    for c in (cache(table_stride=-2),):
        assert L.vafa_paged_decode_workspace(c, 4, 0) == -1
        assert L.vafa_paged_append(c, *app[1:]) == _lib.VAFA_ERR_VALUE
        assert "entries" in _lib.last_error()
