"""Norms with the position rotation, and rows in 8 bits, on the GPU against the 64-bit oracle.

Bounds, element by element (u: half a step of the type relative to a value, 2^-8 bf16, 2^-11
fp16, 2^-24 fp32; a: half the smallest step of fp16, 2^-25; both apply to what is rounded):

* forward: fp32 sums of up to 256 squares in chains of at most 20 additions, so 1 / sqrt(mean)
  is off by 13 fp32 half steps at most, the row by two more products: 15 * 2^-24 < 2^-20; the
  turned pair by 2^-20 (|y1| + |y2|) (sine, cosine and three roundings), with rot_scale's one
  more: together 3 * 2^-20 of the magnitudes, then the output's own rounding u |y| + a.
* dx: g as the turned pair, products and the mean of up to 256 terms: at most 2^-18 of the
  magnitudes that enter, then u |dx| + a.  dweight: the same of every row, and chains of at
  most 256 additions: (2^-18 + 2^-16) of the magnitudes.
* codes: between the roundings of y - d and y + d, d the forward's bound in fp32.
"""
import itertools

import numpy as np
import pytest
import torch

from oracle import head_rows as hr
from oracle import paged as op
from test_gpu_paged import A, U, cache_pair, f64, pages_for, within
from varlenabsorbflashattn_amd import packed_qk_norm_rope, paged_kv_append, paged_kv_gather

pytestmark = pytest.mark.gpu

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
KIND = {torch.bfloat16: "bf16", torch.float16: "fp16"}
FWD, BWD, DW = 3 * 2.0 ** -20, 2.0 ** -18, 2.0 ** -18 + 2.0 ** -16


def freqs(rot):
    return (10000.0 ** (-torch.arange(0, rot, 2) / rot)).float() if rot else None


def dev(t, device):
    return None if t is None else t.to(device)


ROWS = [
    # T, H, Hk, D, rot, interleaved, rot_scale, weights ("" none), dtype
    (1, 1, 1, 64, 64, False, 1.0, "fp32", torch.bfloat16),
    (37, 4, 1, 64, 32, True, 1.0, "same", torch.float16),
    (130, 6, 3, 128, 128, False, 1.25, "fp32", torch.bfloat16),
    (5, 5, 1, 128, 64, False, 0.5, "same", torch.bfloat16),
    (66, 3, 2, 256, 256, True, 1.0, "fp32", torch.float16),
    (1000, 16, 4, 64, 16, False, 1.0, "fp32", torch.bfloat16),
    (19, 2, 2, 256, 0, False, 1.0, "same", torch.bfloat16),
    (700, 32, 8, 128, 128, False, 1.0, "fp32", torch.bfloat16),
    (50, 4, 2, 128, 128, True, 2.0, "", torch.float16),
    (33, 2, 1, 64, 64, False, 1.0, "q", torch.bfloat16),
    (3, 64, 1, 64, 48, False, 1.0, "k", torch.float16),
    (40, 3, 3, 128, 0, False, 1.0, "", torch.bfloat16),
]


def rows_case(case, device):
    T, H, Hk, D, rot, inter, rs, weights, dt = ROWS[case]
    print(f"[rows] {ROWS[case]}", flush=True)
    g = torch.Generator(device=device).manual_seed(case + 1)

    def rnd(*s):
        return torch.randn(*s, generator=g, device=device)
    qkv = rnd(T, H + 2 * Hk, D).to(dt)  # parts of one projection
    w = {n: (1 + 0.3 * rnd(D)).to(dt if weights == "same" else torch.float32) for n in "qk"}
    w = {n: t if weights in ("same", "fp32", n) else None for n, t in w.items()}
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=device, dtype=torch.int32)
    kw = {"positions": pos if rot else None, "inv_freq": dev(freqs(rot), device),
          "interleaved": inter, "rot_scale": rs, "eps": 1e-5}
    return qkv[:, :H], qkv[:, H:H + Hk], w, kw, (rnd(T, H, D).to(dt), rnd(T, Hk, D).to(dt))


@pytest.mark.parametrize("case", range(len(ROWS)))
def test_rows(device, case):
    q, k, w, kw, dy = rows_case(case, device)
    dt = q.dtype
    leaves = [t.detach().requires_grad_(True) for t in (q, k)]
    ws = [None if w[n] is None else w[n].detach().requires_grad_(True) for n in "qk"]
    out = packed_qk_norm_rope(*leaves, q_weight=ws[0], k_weight=ws[1], **kw)
    wants = leaves + [t for t in ws if t is not None]
    grads = list(torch.autograd.grad(out, wants, dy))
    with torch.no_grad():
        again = packed_qk_norm_rope(q, k, q_weight=w["q"], k_weight=w["k"], **kw)
    torch.cuda.synchronize()
    u, a = U[dt], A[dt]
    pos = None if kw["positions"] is None else kw["positions"].cpu().numpy()
    args = (pos, f64(kw["inv_freq"]), kw["interleaved"])
    weight_grads = grads[2:]
    for i, (n, x) in enumerate((("q", q), ("k", k))):
        assert torch.equal(out[i], again[i])
        wn = f64(w[n])
        ref, mag = hr.forward(f64(x), *args, wn, 1e-5, kw["rot_scale"])
        within(n, out[i], ref, FWD * mag + u * np.abs(ref) + a)
        dx, dmag, dw, wmag = hr.backward(f64(x), f64(dy[i]), *args, wn, 1e-5, kw["rot_scale"])
        within("d" + n, grads[i], dx, BWD * dmag + u * np.abs(dx) + a)
        if dw is not None:
            got = weight_grads.pop(0)
            assert got.dtype == w[n].dtype
            uw, aw = (2.0 ** -24, 0.0) if got.dtype == torch.float32 else (u, a)
            within("dw" + n, got, dw, DW * wmag + uw * np.abs(dw) + aw)
    assert not weight_grads


def test_rows_gradients_against_differences(device):
    """Differences of the forward in directions that move every row: in fp32 the products of a
    bf16 forward with dy hold 2^-9 of the sum of |y dy| at worst, and a step of 1/4 moves y by
    far more."""
    q, k, w, kw, dy = rows_case(2, device)
    g = torch.Generator(device=device).manual_seed(99)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, w["q"], w["k"])]
    out = packed_qk_norm_rope(leaves[0], leaves[1], q_weight=leaves[2], k_weight=leaves[3], **kw)
    grads = torch.autograd.grad(out, leaves, dy)
    # the weights enter linearly: differences are exact but for the outputs' rounding
    for i in (2, 3):
        d = torch.randn(leaves[i].shape, generator=g, device=device)
        ys = []
        for s in (0.5, -0.5):
            x = [t.detach().clone() for t in leaves]
            x[i] += s * d
            ys.append(packed_qk_norm_rope(x[0], x[1], q_weight=x[2], k_weight=x[3], **kw)[i - 2])
        want = ((ys[0].double() - ys[1].double()) * dy[i - 2].double()).sum()
        got = (grads[i].double() * d.double()).sum()
        slack = sum((y.double().abs() * dy[i - 2].double().abs()).sum() for y in ys) * U[q.dtype]
        assert abs(got - want) <= slack, (got, want, slack)
        assert abs(got) > 0 and slack < 100 * abs(want) + 1e4


def test_rows_partial_and_missing_gradients(device):
    """Gradients for some of the leaves, and of one output alone."""
    q, k, w, kw, dy = rows_case(3, device)

    def grads(want, use):
        x = {"q": q, "k": k, "qw": w["q"], "kw": w["k"]}
        x = {n: t.detach().requires_grad_(n in want) for n, t in x.items()}
        out = packed_qk_norm_rope(x["q"], x["k"], q_weight=x["qw"], k_weight=x["kw"], **kw)
        return dict(zip(want, torch.autograd.grad([out[i] for i in use], [x[n] for n in want],
                                                  [dy[i] for i in use], allow_unused=True)))
    full = grads(("q", "k", "qw", "kw"), (0, 1))
    for names in (("q",), ("k",), ("qw",), ("kw",), ("q", "kw")):
        for n, t in grads(names, (0, 1)).items():
            assert torch.equal(t, full[n]), (names, n)
    only_q = grads(("q", "k", "qw", "kw"), (0,))
    assert torch.equal(only_q["q"], full["q"]) and torch.equal(only_q["qw"], full["qw"])
    assert not only_q["k"].any() and not only_q["kw"].any()
    # shared by both norms, and q's rows as k's: gradients add up
    x = q.detach().requires_grad_(True)
    s = w["q"].detach().requires_grad_(True)
    out = packed_qk_norm_rope(x, x, q_weight=s, k_weight=s, **kw)
    both = torch.autograd.grad(out, (x, s), (dy[0], dy[0]))
    one = packed_qk_norm_rope(x, x, q_weight=s, k_weight=s, **kw)[0]
    half = torch.autograd.grad(one, (x, s), dy[0])
    assert torch.equal(both[0], half[0] + half[0]) and torch.equal(both[1], half[1] + half[1])


def test_rows_second_derivative_raises(device):
    q, k, w, kw, dy = rows_case(0, device)
    x = q.detach().requires_grad_(True)
    out = packed_qk_norm_rope(x, k.detach(), q_weight=w["q"], **kw)[0]
    g, = torch.autograd.grad(out, x, dy[0], create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        g.sum().backward()


def test_rows_layouts(device):
    """4-D inputs, rows apart from each other, rows that are copied, expanded heads, gradients
    that are not contiguous."""
    q, k, w, kw, dy = rows_case(2, device)
    kw = {**kw, "q_weight": w["q"], "k_weight": w["k"]}
    want = packed_qk_norm_rope(q, k, **kw)
    a, b = packed_qk_norm_rope(q[None], k[None], **kw)
    assert torch.equal(a[0], want[0]) and torch.equal(b[0], want[1])
    T, H, D = q.shape
    odd = torch.zeros(T, H, D + 3, device=device, dtype=q.dtype)
    odd[..., :D] = q
    x = odd[..., :D].detach().requires_grad_(True)
    y, _ = packed_qk_norm_rope(x, k, **kw)
    assert torch.equal(y, want[0])
    far = dy[0].permute(2, 0, 1).contiguous().permute(1, 2, 0)
    g, = torch.autograd.grad(y, x, far)
    z = q.detach().requires_grad_(True)
    g2, = torch.autograd.grad(packed_qk_norm_rope(z, k, **kw)[0], z, dy[0])
    assert torch.equal(g, g2)
    wide = k[:, :1].detach().requires_grad_(True)
    y = packed_qk_norm_rope(wide.expand(T, H, D), k, **kw)[0]
    y2 = packed_qk_norm_rope(k[:, :1].expand(T, H, D).contiguous(), k, **kw)[0]
    assert torch.equal(y, y2)
    g, = torch.autograd.grad(y, wide, dy[0])
    assert g.shape == wide.shape


def test_rows_bad_values_stay_in_their_row(device):
    q, k, w, kw, _ = rows_case(2, device)
    kw = {**kw, "q_weight": w["q"], "k_weight": w["k"]}
    want = packed_qk_norm_rope(q, k, **kw)
    q, k = q.clone(), k.clone()
    q[3, 2, 5], k[7, 1, 100], q[9, 0, 0] = float("inf"), float("nan"), -float("inf")
    got = packed_qk_norm_rope(q, k, **kw)
    bad = [torch.zeros(x.shape[:2], dtype=torch.bool, device=device) for x in want]
    bad[0][3, 2] = bad[0][9, 0] = bad[1][7, 1] = True
    for i in range(2):
        assert torch.equal(got[i][~bad[i]], want[i][~bad[i]])
    assert got[1][7, 1].isnan().all()
    assert got[0][3, 2].isnan().any() and got[0][9, 0].isnan().any()
    # a row of zeros: eps alone keeps it finite
    q.zero_()
    assert not packed_qk_norm_rope(q, k, **kw)[0].any()


def test_rows_empty(device):
    w = torch.ones(64, device=device, requires_grad=True)
    q = torch.zeros(0, 2, 64, device=device, dtype=torch.bfloat16, requires_grad=True)
    pos = torch.zeros(0, dtype=torch.int32, device=device)
    out = packed_qk_norm_rope(q, q[:, :1], pos, inv_freq=freqs(64).to(device), q_weight=w,
                              k_weight=w)
    assert out[0].shape == (0, 2, 64) and out[1].shape == (0, 1, 64)
    gw, = torch.autograd.grad(out[0].sum() + out[1].sum(), w)
    assert gw.shape == (64,) and not gw.any()


def test_rows_many_blocks_repeat(device):
    """Enough rows for every block of the backward to take several runs; the same bits twice,
    and the weights' gradients as sums over parts of the tokens."""
    print("[rows many]", flush=True)
    T, H, Hk, D = 9001, 24, 3, 128
    g = torch.Generator(device=device).manual_seed(77)
    q, dq = (torch.randn(T, H, D, generator=g, device=device).to(torch.bfloat16) for _ in "ab")
    k, dk = (torch.randn(T, Hk, D, generator=g, device=device).to(torch.bfloat16) for _ in "ab")
    w = 1 + 0.1 * torch.randn(2, D, generator=g, device=device)
    pos = torch.arange(T, dtype=torch.int32, device=device)
    inv = freqs(D).to(device)

    def grads(s):
        x = [t.detach().requires_grad_(True) for t in (q[s], k[s], w[0], w[1])]
        out = packed_qk_norm_rope(x[0], x[1], pos[s], inv_freq=inv, q_weight=x[2], k_weight=x[3])
        return torch.autograd.grad(out, x, (dq[s], dk[s]))
    whole, twice = grads(slice(None)), grads(slice(None))
    for a, b in zip(whole, twice):
        assert torch.equal(a, b)
    parts = [grads(slice(i, i + 3001)) for i in range(0, T, 3001)]
    for i in (0, 1):
        assert torch.equal(torch.cat([p[i] for p in parts]), whole[i])
        _, _, dw, mag = hr.backward(f64((q, k)[i]), f64((dq, dk)[i]), pos.cpu().numpy(), f64(inv),
                                    False, f64(w[i]), 1e-6)
        within("dw", whole[2 + i], dw, DW * mag + 2.0 ** -24 * np.abs(dw))


def test_rows_captured(device):
    """A step, forward and backward, in two graphs that share no workspace; replays with other
    values against eager calls."""
    print("[rows graph]", flush=True)
    q, k, w, kw, dy = rows_case(2, device)

    def step(st):
        x = [t.detach().requires_grad_(True) for t in (st["q"], st["k"], st["wq"], st["wk"])]
        out = packed_qk_norm_rope(x[0], x[1], q_weight=x[2], k_weight=x[3], **{**kw, "positions":
                                                                               st["pos"]})
        return [o.detach() for o in out] + list(torch.autograd.grad(out, x, dy))

    def state():
        return {"q": q.clone(), "k": k.clone(), "wq": w["q"].clone(), "wk": w["k"].clone(),
                "pos": kw["positions"].clone()}
    states, graphs = [state(), state()], []
    for st in states:
        step(st)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(st)
        graphs.append((graph, outs))
    g = torch.Generator(device=device).manual_seed(5)
    for i in range(6):
        st, (graph, outs) = states[i % 2], graphs[i % 2]
        for name in ("q", "k", "wq", "wk"):
            st[name].copy_(torch.randn(st[name].shape, generator=g, device=device))
        st["pos"].copy_(torch.randint(0, 5000, st["pos"].shape, generator=g, device=device))
        want = step(st)
        torch.cuda.synchronize()
        for o in outs:
            o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), i


# ---- caches --------------------------------------------------------------------------

def code_caches(g, N, page, Hk, D, device, layout):
    """Two caches of random codes with their powers of two, in one of the layouts."""
    def codes(*s):
        x = torch.randint(0, 256, s, generator=g, device=device).to(torch.uint8)
        return torch.where((x & 127) == 127, x - 1, x).view(E4M3)  # (no NaN)

    def powers(*s):
        return torch.randint(117, 134, s, generator=g, device=device).to(torch.uint8).view(E8M0)
    if layout == "joint":
        c, s = codes(N, 2, page, Hk, D), powers(N, page, 2, Hk)
        return c[:, 0], c[:, 1], s[:, :, 0], s[:, :, 1]
    if layout == "heads":
        return tuple(codes(N, Hk, page, D).transpose(1, 2) for _ in "kv") + \
            tuple(powers(Hk, N, page).permute(1, 2, 0) for _ in "kv")
    return codes(N, page, Hk, D), codes(N, page, Hk, D), powers(N, page, Hk), powers(N, page, Hk)


def values(codes, scale):
    """What a cache of codes stands for, in 64 bits on the host."""
    e = scale.contiguous().view(torch.uint8).cpu().numpy().astype(np.int64) - 127
    return np.ldexp(f64(codes.float()), e[..., None])


APPEND = [
    # lens (None: one token each), past, H, Hk, D, page, rot, inter, rot_scale, weights, codes,
    # dtype, layout
    (None, [0, 1, 15, 16, 500], 4, 2, 64, 16, 64, False, 1.0, True, True, torch.bfloat16, "plain"),
    (None, [7, 100000, 3], 8, 8, 128, 256, 128, False, 1.5, True, True, torch.float16, "joint"),
    ([5, 0, 33, 1], [0, 9, 14, 31], 6, 3, 128, 16, 64, True, 1.0, True, True, torch.bfloat16,
     "heads"),
    ([130, 64], [1, 0], 5, 1, 256, 64, 256, False, 1.0, False, True, torch.float16, "plain"),
    ([3, 20], [2, 4], 2, 2, 64, 7, 16, True, 1.0, True, True, torch.bfloat16, "plain"),
    ([17, 2], [0, 0], 1, 1, 128, 32, 0, False, 1.0, False, True, torch.bfloat16, "plain"),
    ([17, 2], [0, 5], 0, 2, 256, 1, 256, True, 1.0, False, True, torch.float16, "joint"),
    ([40, 90], [3, 8], 4, 2, 128, 16, 128, False, 1.0, True, False, torch.bfloat16, "joint"),
    (None, [30, 0], 4, 1, 64, 16, 32, True, 0.7, True, False, torch.float16, "heads"),
    ([1] * 130, [i * 3 for i in range(130)], 2, 1, 64, 16, 32, False, 1.0, True, True,
     torch.bfloat16, "plain"),
    ([700, 1, 333], [50, 0, 1], 32, 8, 128, 64, 128, False, 1.0, True, True, torch.bfloat16,
     "plain"),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_store(device, case):
    lens, past, H, Hk, D, page, rot, inter, rs, weights, codes, dt, layout = APPEND[case]
    print(f"[store] {APPEND[case]}", flush=True)
    g = torch.Generator(device=device).manual_seed(case + 41)
    new = [1] * len(past) if lens is None else lens
    T, extra = sum(new), 0 if lens is None else 5  # rows behind the last sequence
    qkv = torch.randn(T + extra, H + 2 * Hk, D, generator=g, device=device)
    # rows of very unequal sizes
    qkv *= 2.0 ** torch.randint(-9, 9, qkv.shape[:2], generator=g, device=device)[..., None]
    qkv = qkv.to(dt)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    table, N = pages_for(g, [a + b for a, b in zip(new, past)], page)
    if codes:
        kc, vc, ks, vs = code_caches(g, N, page, Hk, D, device, layout)
        kw = {"k_scale": ks, "v_scale": vs}
        old = [values(kc, ks), values(vc, vs)]
    else:
        kc, vc = cache_pair(g, N, page, Hk, D, dt, device, layout)
        kw, ks, vs = {}, None, None
        old = [f64(kc), f64(vc)]
    before = [t.clone() for t in (kc.view(torch.uint8), vc.view(torch.uint8))] if codes else None
    w = [1 + 0.3 * torch.randn(D, generator=g, device=device) for _ in "qk"] if weights \
        else [None, None]
    if H:
        kw.update(q=q, q_weight=w[0])
    cu = None if lens is None else torch.tensor(np.cumsum([0] + new), dtype=torch.int32)
    inv = freqs(rot)
    plens = torch.tensor(past, dtype=torch.int32)
    versions = kc._version, vc._version
    out = paged_kv_append(k, v, kc, vc, table.to(device), plens.to(device),
                          cu_seqlens=dev(cu, device), inv_freq=dev(inv, device), interleaved=inter,
                          k_weight=w[1], eps=1e-5, rot_scale=rs, **kw)
    torch.cuda.synchronize()
    assert kc._version > versions[0] and vc._version > versions[1]
    u, a, kind = U[dt], A[dt], KIND[dt]
    hcu = np.arange(len(new) + 1) if cu is None else cu.numpy()
    pos, seq = np.zeros(T, np.int64), np.zeros(T, np.int64)
    for b in range(len(new)):
        pos[hcu[b]:hcu[b + 1]] = past[b] + np.arange(new[b])
        seq[hcu[b]:hcu[b + 1]] = b
    args = (pos, f64(inv), inter)
    if H:
        ref, mag = hr.forward(f64(q)[:T], *args, f64(w[0]), 1e-5, rs)
        within("q", out[:T], ref, FWD * mag + u * np.abs(ref) + a)
        assert not out[T:].any()
    else:
        assert out is None
    yk, kmag = hr.forward(f64(k)[:T], *args, f64(w[1]), 1e-5, rs)
    at = [op.place(table.numpy(), N, page, seq[t], pos[t]) for t in range(T)]
    assert all(x is not None for x in at)
    idx = tuple(np.array(x) for x in zip(*at))
    touched = np.zeros((N, page), bool)
    touched[idx] = True
    d = FWD * kmag if (rot or weights) else 0.0 * kmag
    for name, cache, scale, y, dy, o in (("k", kc, ks, yk, d, old[0]),
                                         ("v", vc, vs, f64(v)[:T], 0.0 * yk, old[1])):
        got = values(cache, scale) if codes else f64(cache)
        assert np.array_equal(got[~touched], o[~touched]), name
        if not codes:
            within(name, cache[torch.from_numpy(idx[0]), torch.from_numpy(idx[1])], y,
                   dy + (u * np.abs(y) + a) * (name == "k"))
            continue
        e = scale.contiguous().view(torch.uint8).cpu().numpy().astype(np.int64)[idx] - 127
        amax, off = np.abs(y).max(-1), dy.max(-1)
        low, high = hr.exponent(np.maximum(amax - off, 0.0), kind), hr.exponent(amax + off, kind)
        assert (low <= e).all() and (e <= high).all(), name
        val = got[idx]
        assert (val >= hr.to_code(y - dy, e[..., None], kind)).all(), name
        assert (val <= hr.to_code(y + dy, e[..., None], kind)).all(), name
    if codes:
        for t, b in zip((kc.view(torch.uint8), vc.view(torch.uint8)), before):
            assert torch.equal(t[torch.from_numpy(~touched).to(device)],
                               b[torch.from_numpy(~touched).to(device)])


def test_store_extreme_values(device):
    """The largest and smallest numbers of the types, zeros, infinities and NaN, ties."""
    for dt in (torch.bfloat16, torch.float16):
        print(f"[store extremes] {dt}", flush=True)
        D, kind, big = 64, KIND[dt], torch.finfo(dt).max
        tiny = torch.finfo(dt).smallest_normal
        rows = torch.zeros(12, D)
        rows[1, :3] = torch.tensor([big, -big, 1.0])
        rows[2, :4] = torch.tensor([float("inf"), 3.0, -1.0, float("nan")])
        rows[3, :2] = torch.tensor([tiny, -tiny / 4])
        rows[4, :2] = torch.tensor([448.0, 450.0])
        rows[5, :3] = torch.tensor([448.0, 17.0, 19.0])      # ties to even at a step of 2
        rows[6, :4] = torch.tensor([1.75, 2.0 ** -16, 3 * 2.0 ** -18, 2.0 ** -18])  # subnormal
        rows[7] = float("nan")
        rows[8] = -float("inf")
        rows[9, :2] = torch.tensor([big / 2, big * 0.93])
        rows[10] = torch.arange(D) * 2.0 ** -7 + 1.0
        rows[11, 0] = -1.7578125  # just past 448 / 256
        x = rows[:, None].to(dt).to(device)
        kc = torch.zeros(1, 16, 1, D, device=device).to(E4M3)
        vc = torch.zeros(1, 16, 1, D, device=device).to(E4M3)
        ks, vs = (torch.zeros(1, 16, 1, dtype=torch.uint8, device=device).view(E8M0) for _ in "kv")
        table = torch.zeros(1, 1, dtype=torch.int32, device=device)
        zero = torch.zeros(1, dtype=torch.int32, device=device)
        cu = torch.tensor([0, 12], dtype=torch.int32, device=device)
        paged_kv_append(x, x, kc, vc, table, zero, cu_seqlens=cu, k_scale=ks, v_scale=vs)
        y = f64(x)[:, 0]
        e = hr.row_exponents(y, kind)
        want = hr.to_code(y, e[:, None], kind)
        for c, s in ((kc, ks), (vc, vs)):
            got = values(c, s)[0, :12, 0]
            assert np.array_equal(s.view(torch.uint8).cpu().numpy()[0, :12, 0] - 127.0, e)
            assert np.array_equal(got, want, equal_nan=True)
        k, v = paged_kv_gather(kc, vc, table, cu, 12, k_scale=ks, v_scale=vs, dtype=dt)
        ref = torch.from_numpy(want).to(dt)
        for t in (k, v):
            assert torch.equal(t[:, 0].cpu().nan_to_num(7.0), ref.nan_to_num(7.0))
            assert torch.equal(t[:, 0].cpu().isnan(), ref.isnan())
            assert not t.isinf().any()


GATHER = [
    # cache lens, starts (None: 0), lens read, Hk, D, page, codes, dtype, layout
    ([5, 0, 70], None, [5, 0, 70], 2, 64, 16, True, torch.bfloat16, "plain"),
    ([100, 33], [7, 30], [60, 3], 3, 128, 7, True, torch.float16, "joint"),
    ([100, 33], [7, 30], [60, 3], 1, 256, 32, True, torch.bfloat16, "heads"),
    ([12, 900], [0, 1], [12, 899], 8, 128, 64, False, torch.bfloat16, "joint"),
    ([12, 90], [0, 1], [12, 89], 1, 80, 1, False, torch.float16, "heads"),
    ([40, 40], None, [40, 40], 2, 48, 16, True, torch.float16, "plain"),
]


@pytest.mark.parametrize("case", range(len(GATHER)))
def test_gather(device, case):
    lens, starts, read, Hk, D, page, codes, dt, layout = GATHER[case]
    print(f"[gather] {GATHER[case]}", flush=True)
    g = torch.Generator(device=device).manual_seed(case + 61)
    table, N = pages_for(g, lens, page)
    if codes:
        kc, vc, ks, vs = code_caches(g, N, page, Hk, D, device, layout)
        kw, vals = {"k_scale": ks, "v_scale": vs, "dtype": dt}, (values(kc, ks), values(vc, vs))
    else:
        kc, vc = cache_pair(g, N, page, Hk, D, dt, device, layout)
        kw, vals = {}, (f64(kc), f64(vc))
    cu = np.cumsum([2] + read)  # two rows in front, three behind
    total = int(cu[-1]) + 3
    st = None if starts is None else torch.tensor(starts, dtype=torch.int32, device=device)
    k, v = paged_kv_gather(kc, vc, table.to(device),
                           torch.tensor(cu, dtype=torch.int32, device=device), total, starts=st,
                           **kw)
    want = hr.gather(*vals, table.numpy(), cu, starts or [0] * len(read), total)
    for t, r in zip((k, v), want):
        assert t.dtype == dt and t.shape == (total, Hk, D)
        assert torch.equal(t.cpu(), torch.from_numpy(r).to(dt))
    # bad pages, positions outside the table, negative starts: zeros
    bad = table.clone()
    bad[0, 0], bad[-1, -1] = N, -3
    far = torch.tensor([-1, 2 ** 31 - 5], dtype=torch.int32, device=device)
    cu2 = torch.tensor([0, 9, 18], dtype=torch.int32, device=device)
    k, v = paged_kv_gather(kc, vc, bad[:2].to(device), cu2, 18, starts=far, **kw)
    want = hr.gather(*vals, bad[:2].numpy(), [0, 9, 18], [-1, 2 ** 31 - 5], 18)
    for t, r in zip((k, v), want):
        assert torch.equal(t.cpu(), torch.from_numpy(r).to(dt))


def test_all_codes_come_back(device):
    """Every code under powers of two from the least to the largest, in both types."""
    print("[all codes]", flush=True)
    codes = torch.arange(256, dtype=torch.uint8)
    kc = codes.view(1, 1, 1, 256).repeat(1, 256, 1, 1).to(device).view(E4M3)
    e = torch.arange(256, dtype=torch.uint8).clamp(max=254).view(1, 256, 1).to(device)
    table = torch.zeros(1, 1, dtype=torch.int32, device=device)
    cu = torch.tensor([0, 256], dtype=torch.int32, device=device)
    want = np.ldexp(f64(kc.float())[0, :, 0], e.cpu().numpy()[0].astype(np.int64) - 127)
    for dt in (torch.bfloat16, torch.float16):
        k, v = paged_kv_gather(kc, kc, table, cu, 256, k_scale=e.view(E8M0), v_scale=e.view(E8M0),
                               dtype=dt)
        assert torch.equal(k.nan_to_num(7.0), v.nan_to_num(7.0))
        ref = torch.from_numpy(want).to(dt)
        # (rows that an append writes: from 2^-126 on, and finite in their type)
        some = torch.from_numpy(np.isfinite(want)) & ref.isfinite()
        some[0] = False
        got = k[:, 0].cpu()
        assert torch.equal(got[some], ref[some])
        assert got[1:255, [127, 255]].isnan().all()


def test_append_and_gather_follow_the_packed_rows(device):
    """As they would be used together: what packed_qk_norm_rope gives training is what the
    cache of a prompt holds, in 16 bits to the bit, in 8 bits after its rounding."""
    print("[serve as trained]", flush=True)
    dt, H, Hk, D, page = torch.bfloat16, 8, 2, 128, 16
    g = torch.Generator(device=device).manual_seed(3)
    lens, past = [33, 1, 90], [0, 20, 7]
    T = sum(lens)
    x = torch.randn(T, H + 2 * Hk, D, generator=g, device=device).to(dt)
    q, k, v = x[:, :H], x[:, H:H + Hk], x[:, H + Hk:]
    w = 1 + 0.1 * torch.randn(2, D, generator=g, device=device)
    inv = freqs(D).to(device)
    pos = torch.cat([p + torch.arange(n) for n, p in zip(lens, past)]).int().to(device)
    kw = {"inv_freq": inv, "q_weight": w[0], "k_weight": w[1], "rot_scale": 1.1}
    yq, yk = packed_qk_norm_rope(q, k, pos, **kw)
    table, N = pages_for(g, [a + b for a, b in zip(lens, past)], page)
    table = table.to(device)
    cu = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=device)
    plens = torch.tensor(past, dtype=torch.int32, device=device)
    kc, vc = cache_pair(g, N, page, Hk, D, dt, device, "plain")
    out = paged_kv_append(k, v, kc, vc, table, plens, cu_seqlens=cu, q=q, **kw)
    gk, gv = paged_kv_gather(kc, vc, table, cu, T, starts=plens)
    assert torch.equal(out, yq) and torch.equal(gk, yk) and torch.equal(gv, v)
    kc, vc, ks, vs = code_caches(g, N, page, Hk, D, device, "plain")
    out = paged_kv_append(k, v, kc, vc, table, plens, cu_seqlens=cu, q=q, k_scale=ks, v_scale=vs,
                          **kw)
    gk, gv = paged_kv_gather(kc, vc, table, cu, T, starts=plens, k_scale=ks, v_scale=vs, dtype=dt)
    assert torch.equal(out, yq)
    for got, ref in ((gk, f64(yk)), (gv, f64(v))):
        e = hr.row_exponents(ref, "bf16")[..., None]
        # half a step of e4m3, and of bf16 where the packed rows were rounded before
        assert (np.abs(f64(got) - ref) <= (2.0 ** -4 + 2.0 ** -7) * np.abs(ref)
                + np.ldexp(1.0, e - 9)).all()


def test_codes_under_graph_capture(device):
    """Storing and reading back in a graph, replayed with other tokens, lengths and pages."""
    print("[codes graph]", flush=True)
    dt, H, Hk, D, page, n = torch.bfloat16, 4, 2, 64, 16, 3
    g = torch.Generator(device=device).manual_seed(19)
    kc, vc, ks, vs = code_caches(g, 30, page, Hk, D, device, "plain")
    x = torch.zeros(n, H + 2 * Hk, D, device=device, dtype=dt)
    table = torch.zeros(n, 10, dtype=torch.int32, device=device)
    lens = torch.zeros(n, dtype=torch.int32, device=device)
    cu = torch.arange(n + 1, dtype=torch.int32, device=device)
    w, inv = torch.ones(D, device=device), freqs(D).to(device)

    def step(caches):
        kc, vc, ks, vs = caches
        q = paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], kc, vc, table, lens, q=x[:, :H],
                            inv_freq=inv, q_weight=w, k_weight=w, k_scale=ks, v_scale=vs)
        return (q,) + paged_kv_gather(kc, vc, table, cu, n, starts=lens, k_scale=ks, v_scale=vs,
                                      dtype=dt)
    step((kc, vc, ks, vs))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step((kc, vc, ks, vs))
    for i in range(5):
        x.copy_(torch.randn(x.shape, generator=g, device=device))
        table.copy_(torch.randperm(30, generator=g, device=device).view(n, 10))
        lens.copy_(torch.tensor([17 * i % 160, i, 159], dtype=torch.int32))
        other = [t.clone() for t in (kc, vc, ks.view(torch.uint8), vs.view(torch.uint8))]
        want = step((other[0], other[1], other[2].view(E8M0), other[3].view(E8M0)))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), i
        for a, b in zip((kc, vc, ks, vs), other):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), i


def test_codes_past_4_gib(device):
    """Codes beyond 4 GiB of a cache, and scales of theirs."""
    page, Hk, D, dt = 256, 2, 128, torch.bfloat16
    N = (5 << 30) // (page * Hk * D)
    print(f"[far codes] {N} pages", flush=True)
    g = torch.Generator(device=device).manual_seed(12)
    kc = torch.zeros(N, page, Hk, D, device=device, dtype=torch.uint8).view(E4M3)
    vc = torch.zeros(N, page, Hk, D, device=device, dtype=torch.uint8).view(E4M3)
    ks, vs = (torch.zeros(N, page, Hk, device=device, dtype=torch.uint8).view(E8M0) for _ in "kv")
    x = torch.randn(700, 2 * Hk, D, generator=g, device=device).to(dt)
    cu = torch.tensor([0, 700], dtype=torch.int32, device=device)
    zero = torch.zeros(1, dtype=torch.int32, device=device)
    outs = []
    for pages in ([0, 1, 2], [N - 1, N - 3, N - 2]):
        table = torch.tensor([pages], dtype=torch.int32, device=device)
        paged_kv_append(x[:, :Hk], x[:, Hk:], kc, vc, table, zero, cu_seqlens=cu, k_scale=ks,
                        v_scale=vs)
        outs.append(paged_kv_gather(kc, vc, table, cu, 700, k_scale=ks, v_scale=vs, dtype=dt))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and a.any()
    assert not kc.view(torch.uint8)[3:N - 3].any()


def test_codes_streams(device):
    """Work queued on another stream than the tensors' own."""
    print("[codes streams]", flush=True)
    q, k, w, kw, dy = rows_case(2, device)
    kw = {**kw, "q_weight": w["q"], "k_weight": w["k"]}
    want = packed_qk_norm_rope(q, k, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for s in itertools.islice(itertools.cycle((side, torch.cuda.current_stream())), 4):
        with torch.cuda.stream(s):
            outs.append(packed_qk_norm_rope(q, k, **kw))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


# Rows of bf16 whose squares leave fp32 on either side: eps and the rows' sizes.
EXTREME = [
    (1e-6, [1.0, 1e19, 2e20, 1e30, 2.0 ** 126]),
    (0.0, [1.0, 1e20, 1e-19, 1e-25, 2.0 ** -120, 2.0 ** -131]),
    (2.0 ** -100, [1e-15, 3e-16, 1e-20, 1e-10, 1e-30, 1e25]),
]


@pytest.mark.parametrize("D,inter", [(64, False), (128, True), (256, False)])
@pytest.mark.parametrize("eps,sizes", EXTREME)
def test_rows_of_extreme_sizes(device, D, inter, eps, sizes):
    """Sums of squares that pass 2^127 or fall below 2^-149 in fp32 are formed of rows scaled by a
    power of two, which rounds nothing (features of a row are within 2^24 of each other here): the
    bounds are those of ordinary rows.  dy is scaled so that dx stays a normal number."""
    print(f"[rows extreme] D {D} eps {eps} {sizes}", flush=True)
    g = torch.Generator(device=device).manual_seed(D)
    H, Hk, n = 3, 2, 40
    size = torch.tensor(sizes, device=device, dtype=torch.float64).repeat(n)
    T = len(size)

    def rows(h, s):
        x = torch.randn(T, h, D, generator=g, device=device).clamp(-1.9, 1.9)
        return (x.double() * s[:, None, None]).to(torch.bfloat16)
    q, k = rows(H, size), rows(Hk, size)
    assert q.isfinite().all() and k.isfinite().all()
    dy = [rows(h, size.clamp(2.0 ** -20, 2.0 ** 20)) for h in (H, Hk)]
    w = 1 + 0.3 * torch.randn(2, D, generator=g, device=device)
    pos = torch.arange(T, dtype=torch.int32, device=device)
    inv = freqs(D).to(device)
    kw = {"inv_freq": inv, "interleaved": inter, "eps": eps}
    leaves = [t.detach().requires_grad_(True) for t in (q, k, w[0], w[1])]
    out = packed_qk_norm_rope(leaves[0], leaves[1], pos, q_weight=leaves[2], k_weight=leaves[3],
                              **kw)
    grads = torch.autograd.grad(out, leaves, dy)
    u, args = U[q.dtype], (pos.cpu().numpy(), f64(inv), inter)
    for i, x in enumerate((q, k)):
        ref, mag = hr.forward(f64(x), *args, f64(w[i]), eps)
        within("qk"[i], out[i], ref, FWD * mag + u * np.abs(ref))
        dx, dmag, dw, wmag = hr.backward(f64(x), f64(dy[i]), *args, f64(w[i]), eps)
        within("d" + "qk"[i], grads[i], dx, BWD * dmag + u * np.abs(dx))
        within("dw", grads[2 + i], dw, DW * wmag + 2.0 ** -24 * np.abs(dw))
    # the same on the way into caches of both kinds
    table = torch.zeros(1, 1, dtype=torch.int32, device=device)
    zero, cu = table[0, :1].clone(), torch.tensor([0, T], dtype=torch.int32, device=device)
    append = {"cu_seqlens": cu, "q": q, "q_weight": w[0], "k_weight": w[1], **kw}
    kc, vc = torch.zeros(2, 1, T, Hk, D, device=device, dtype=q.dtype)
    assert torch.equal(paged_kv_append(k, k, kc, vc, table, zero, **append), out[0])
    assert torch.equal(kc[0], out[1]) and torch.equal(vc[0], k)
    kc, vc = (torch.zeros(1, T, Hk, D, device=device).to(E4M3) for _ in "kv")
    ks, vs = (torch.zeros(1, T, Hk, dtype=torch.uint8, device=device).view(E8M0) for _ in "kv")
    got = paged_kv_append(k, k, kc, vc, table, zero, k_scale=ks, v_scale=vs, **append)
    assert torch.equal(got, out[0])
    y, off = ref, (FWD * mag).max(-1)
    e = ks.view(torch.uint8).cpu().numpy()[0].astype(np.int64) - 127
    amax = np.abs(y).max(-1)
    assert (hr.exponent(np.maximum(amax - off, 0.0), "bf16") <= e).all()
    assert (e <= hr.exponent(amax + off, "bf16")).all()
    val = values(kc, ks)[0]
    assert (val >= hr.to_code(y - FWD * mag, e[..., None], "bf16")).all()
    assert (val <= hr.to_code(y + FWD * mag, e[..., None], "bf16")).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rot,inter", [(0, False), (64, False), (64, True), (32, False)])
def test_rows_with_infinities_and_nan(device, dt, rot, inter):
    """What an infinity or NaN does to its row: normed, the mean is infinite, so features are 0,
    and NaN where the infinity stands (inf / inf) and at the other of its pair; a NaN takes the
    whole row.  Rows without a weight are not normed: pairs that hold neither stay."""
    print(f"[rows inf] {dt} rot {rot} {inter}", flush=True)
    D, H, n = 64, 2, rot // 2
    g = torch.Generator(device=device).manual_seed(rot)
    x = torch.randn(7, H, D, generator=g, device=device).to(dt)
    k = torch.randn(7, 1, D, generator=g, device=device).to(dt)
    w = 1 + 0.1 * torch.rand(D, generator=g, device=device)
    pos = 3 + torch.arange(7, dtype=torch.int32, device=device)
    kw = {"inv_freq": dev(freqs(rot), device), "interleaved": inter}
    plain = packed_qk_norm_rope(x, k, pos, **kw)[0]
    normed = packed_qk_norm_rope(x, k, pos, q_weight=w, k_weight=w, **kw)
    bad = x.clone()
    places = [(1, 0, 5), (2, 1, 40), (4, 0, 63)]
    for (t, h, i), value in zip(places, (float("inf"), -float("inf"), float("inf"))):
        bad[t, h, i] = value
    bad[5, 1, 9] = float("nan")

    def pair(i):
        if i >= rot:
            return {i}
        return {i, i ^ 1} if inter else {i, (i + n) % rot}
    leaf, weight = bad.detach().requires_grad_(True), w.detach().requires_grad_(True)
    out, kout = packed_qk_norm_rope(leaf, k, pos, q_weight=weight, k_weight=w, **kw)
    dx, dw = torch.autograd.grad(out, (leaf, weight), torch.ones_like(out))
    bare = packed_qk_norm_rope(bad, k, pos, **kw)[0]
    assert torch.equal(kout, normed[1])
    good = torch.ones(7, H, dtype=torch.bool, device=device)
    for t, h, i in places:
        good[t, h] = False
        at = torch.zeros(D, dtype=torch.bool, device=device)
        at[list(pair(i))] = True
        assert out[t, h][at].isnan().all() and not out[t, h][~at].any()
        assert torch.equal(bare[t, h][~at], plain[t, h][~at])
        assert not bare[t, h][at].isfinite().any()
        assert i < rot or bare[t, h, i] == bad[t, h, i]
        assert dx[t, h].isnan().all() and dw[i].isnan()
    good[5, 1] = False
    assert out[5, 1].isnan().all() and dx[5, 1].isnan().all() and dw.isnan().all()
    assert torch.equal(out[good], normed[0][good]) and dx[good].isfinite().all()
    # zeros: eps alone keeps a normed row finite
    zero = torch.zeros_like(x)
    for eps, nan in ((1e-45, False), (1e-30, False), (0.0, True)):
        got = packed_qk_norm_rope(zero, k, pos, q_weight=w, k_weight=w, eps=eps, **kw)[0]
        assert got.isnan().all() if nan else not got.any()
