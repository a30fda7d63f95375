"""Packed attention under a mask, on the CPU: the plan covers exactly what the mask lets
through, the calls that are refused, and the oracle against torch and differences."""
import math

import numpy as np
import pytest
import torch

from oracle import masked as om
from varlenabsorbflashattn_amd import _lib, packed_masked_attn


def cu(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


def walked(item, window, bn):
    """Keys that a kernel walks for a forward item (key_walk in csrc/masked.h)."""
    q0, q1, k0, k1, _, diag, pre, _ = (int(x) for x in item)
    win0 = q0 + diag - window + 1
    a1, wl = min(pre, k1), max(win0, k0)
    if a1 > k0:
        if wl > a1:
            return list(range(k0, a1)) + list(range(wl, k1))
        return list(range(k0, k1))
    return list(range(wl, k1))


CASES = [
    # q lens, k lens, H, Hk, D, causal, window, prefix
    ([5, 0, 300, 129], [5, 0, 300, 129], 4, 2, 64, True, 0, None),
    ([5, 40, 7], [1, 900, 0], 4, 4, 128, True, 0, None),          # rows without keys
    ([700, 33], [700, 1200], 2, 1, 128, True, 50, None),
    ([700, 33, 1], [700, 1200, 4000], 8, 2, 256, True, 64, [100, 1200, 3]),
    ([260, 10], [300, 10], 3, 3, 64, True, 0, [300, 0]),
    ([130, 1], [70, 5000], 2, 2, 128, False, 0, None),
    ([1, 16], [20000, 9000], 1, 1, 128, True, 0, None),            # split over keys
    ([300], [9000], 2, 1, 64, True, 2500, [700]),                  # split across the gap
    ([2, 1], [0, 0], 1, 1, 64, True, 0, None),
    ([70, 3000, 9], [70, 3000, 40], 24, 2, 128, True, 0, None),    # sets of 4 heads, parts
    ([2000], [2000], 64, 1, 256, True, 300, [100]),                # sets of 32, parts
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_plan_covers_the_mask(case):
    ql, kl, H, Hk, D, causal, window, prefix = CASES[case]
    cq, ck = cu(ql), cu(kl)
    p = _lib.plan_masked(cq, ck, H, Hk, D, causal, window, prefix)
    info, win = p.info, window or 1 << 30
    assert (info.T_q, info.T_k, info.H, info.kind) == (cq[-1], ck[-1], H, 3)
    sets = 1 << info.xcd_heads  # heads in the rows of a tile
    assert (H // Hk) % sets == 0 and sets <= 32 and (sets == 32 or (H // Hk) % (2 * sets) != 0)
    see = np.zeros((cq[-1], ck[-1]), bool)
    for s in range(len(ql)):
        see[cq[s]:cq[s + 1], ck[s]:ck[s + 1]] = om.visible(
            ql[s], kl[s], causal, window, prefix[s] if prefix else 0)
    seg = np.searchsorted(cq, np.arange(cq[-1]), side="right") - 1
    for items, sums, tile in (("fwd", "comb", info.q_tile), ("dq", "dqc", 128)):
        got = np.zeros(see.shape, int)
        owners = np.zeros(cq[-1], int)
        prows = set()
        for it in p.section(items):
            q0, q1, k0, k1, pbase, diag, pre, owner = (int(x) for x in it)
            assert 0 <= q0 < q1 <= cq[-1] and 0 <= k0 <= k1 <= ck[-1] and (q1 - q0) * sets <= tile
            assert len(set(seg[q0:q1])) == 1
            s = seg[q0]
            assert diag == ck[s + 1] - cq[s + 1] and ck[s] <= k0 and k1 <= ck[s + 1]
            assert pre == (ck[s + 1] if not causal else ck[s] + (prefix[s] if prefix else 0))
            owners[q0:q1] += owner
            if pbase >= 0:
                rows = set(range(pbase, pbase + q1 - q0))
                assert not rows & prows and pbase + q1 - q0 <= info.n_part_rows
                prows |= rows
            got[q0:q1, walked(it, win, 64)] += 1
        assert (owners == 1).all()
        assert got.max(initial=0) <= 1 and (got[see] == 1).all()
        # the sums read exactly the split items' rows
        read = set()
        for q0, q1, pbase, ns, *_ in p.section(sums).tolist():
            rows = set(range(pbase, pbase + ns * (q1 - q0)))
            assert not rows & read
            read |= rows
        assert read == prows and len(prows) <= info.n_part_rows
    # every key once, or by all the parts of its tile, which own the rows that are summed
    keys, prows, parts_of = np.zeros(ck[-1]), {}, {}
    for it in p.section("kv"):
        k0, k1, q0, q1, diag, pre, pbase, part = (int(x) for x in it)
        part, parts = part >> 16, part & 0xffff
        assert 0 <= k0 < k1 <= ck[-1] and 0 <= q0 <= q1 <= cq[-1] and k1 - k0 <= info.k_tile
        assert 0 <= part < parts and (pbase >= 0) == (parts > 1)
        keys[k0:k1] += 1.0 / parts
        parts_of.setdefault(k0, []).append((part, parts, pbase, k1 - k0))
        rows = np.zeros(cq[-1], bool)
        rows[q0:q1] = True
        assert not see[~rows, k0:k1].any()
        assert (seg[q0:q1] == np.searchsorted(ck, k0, side="right") - 1).all()
    np.testing.assert_allclose(keys, 1.0)
    sums = {k0: (k1, pbase, n) for k0, k1, pbase, n, *_ in p.section("fcomb").tolist()}
    used = set()
    for k0, got in parts_of.items():
        got.sort()
        assert [g[0] for g in got] == list(range(got[0][1]))
        if got[0][1] == 1:
            assert k0 not in sums
            continue
        k1, pbase, n = sums.pop(k0)
        assert n == got[0][1] and k1 - k0 == got[0][3]
        for part, _, at, rows in got:
            assert at == pbase + part * rows
            new = set(range(at, at + rows))
            assert not new & used
            used |= new
    assert not sums and len(used) == info.n_fpart_rows


def test_plan_refusals():
    c = cu([4, 4])

    def bad(error, text, *args, **kw):
        with pytest.raises(error, match=text):
            _lib.plan_masked(c, c, *args, **kw)
    bad(AssertionError, "do not divide", 3, 2, 64)
    bad(AssertionError, "do not divide", 0, 1, 64)
    bad(ValueError, "more than 4096 query heads", 8192, 8, 64)
    bad(ValueError, "belong to the causal", 2, 1, 64, False, 5)
    bad(ValueError, "belong to the causal", 2, 1, 64, False, 0, [1, 1])
    bad(ValueError, "window must be positive", 2, 1, 64, True, -1)
    bad(ValueError, r"prefix_lens\[1\] = 5 of 4", 2, 1, 64, True, 0, [4, 5])
    bad(ValueError, r"prefix_lens\[0\] = -1", 2, 1, 64, True, 0, [-1, 0])
    assert _lib.plan_masked(c, c, 40, 1, 64).info.xcd_heads == 3
    bad(AssertionError, "prefix_lens must be", 2, 1, 64, True, 0, [1])
    big = np.array([0, (1 << 30) + 1])
    with pytest.raises(ValueError, match="more than"):
        _lib.plan_masked(big, big, 1, 1, 64)


def test_c_abi_refusals():
    import ctypes as C
    L = _lib.lib()
    p = _lib.plan_masked(cu([4]), cu([4]), 4, 2, 64)
    other = _lib.plan_varlen(cu([4]), cu([4]), 4, 64)
    assert L.vafa_masked_fwd_workspace(other.info, 2, 64) == -1
    assert L.vafa_masked_bwd_workspace(p.info, 3, 64) == -1
    assert L.vafa_masked_bwd_workspace(p.info, 1, 64) == -1  # built for other sets of heads
    assert L.vafa_masked_bwd_workspace(p.info, 2, 96) == -1
    assert L.vafa_varlen_fwd_workspace(p.info, 64) == -1  # and not the other way round
    need = L.vafa_masked_bwd_workspace(p.info, 2, 64)
    assert need > 0
    x = 1 << 20
    f = [x, x, x, x, x, x, x, p.info, 2, 64, _lib.DT_BF16, 0.1, 0.0, 0, None, x, 1 << 20, None]
    b = [x] * 11 + [p.info, 2, 64, _lib.DT_BF16, 0.1, 0.0, 0, None, x, need, None]

    def rc(call, args, at, value):
        return call(*[value if i == at else y for i, y in enumerate(args)])
    for at, bad, want in ((0, x + 2, "VALUE"), (8, 3, "ASSERT"), (9, 32, "ASSERT"),
                          (10, _lib.DT_F32, "ASSERT"), (11, float("nan"), "VALUE"),
                          (11, 3e38, "VALUE"), (12, -2.0, "VALUE"), (12, 1e-40, "VALUE"),
                          (12, 3e5, "VALUE"), (13, -1, "VALUE"), (7, other.info, "VALUE")):
        assert rc(L.vafa_masked_fwd, f, at, bad) == getattr(_lib, "VAFA_ERR_" + want), at
    for at, bad, want in ((5, x + 8, "VALUE"), (4, None, "VALUE"), (20, need - 1, "WORKSPACE"),
                          (19, None, "WORKSPACE"), (19, x + 4, "WORKSPACE"),
                          (16, float("inf"), "VALUE")):
        assert rc(L.vafa_masked_bwd, b, at, bad) == getattr(_lib, "VAFA_ERR_" + want), at
    assert C.sizeof(_lib.PagedCache) == 17 * 8


def _call(dt=torch.bfloat16, H=4, Hk=2, D=64, **kw):
    q, k = torch.zeros(6, H, D, dtype=dt), torch.zeros(6, Hk, D, dtype=dt)
    c = torch.tensor([0, 6], dtype=torch.int32)
    kw = {"cu_seqlens_q": c, "cu_seqlens_k": c, **kw}
    return packed_masked_attn(q, k, kw.pop("v", k), **kw)


def test_call_refusals():
    slopes = torch.ones(4)
    for kw, error, text in (
            ({"dt": torch.float32}, AssertionError, "dtype"),
            ({"D": 96}, AssertionError, "head_dim 96"),
            ({"H": 3}, AssertionError, "do not divide"),
            ({"v": torch.zeros(6, 2, 64)}, AssertionError, "share dtype"),
            ({"v": torch.zeros(5, 2, 64, dtype=torch.bfloat16)}, AssertionError, "T_k, H_k"),
            ({"v": torch.zeros(6, 128, dtype=torch.bfloat16)}, ValueError, "got 2-D"),
            ({"v": torch.zeros(2, 6, 2, 64, dtype=torch.bfloat16)}, ValueError, "batch=1"),
            ({"alibi_slopes": slopes.double()}, AssertionError, "alibi_slopes"),
            ({"alibi_slopes": slopes[:3]}, AssertionError, "alibi_slopes"),
            ({"alibi_slopes": slopes.clone().requires_grad_(True)}, ValueError, "no gradient"),
            ({}, AssertionError, "requires GPU tensors")):
        with pytest.raises(error, match=text):
            _call(**kw)


def test_option_refusals():
    from varlenabsorbflashattn_amd import masked
    c = torch.tensor([0, 6], dtype=torch.int32)
    for kw, error, text in (
            ({"window": 0}, ValueError, "window must be positive"),
            ({"softcap": -1.0}, ValueError, "softcap"),
            ({"softcap": 0.0}, ValueError, "softcap"),
            ({"softcap": float("inf")}, ValueError, "softcap"),
            ({"softcap": 1e-50}, ValueError, "softcap"),
            ({"softcap": 2e4}, ValueError, "softcap"),
            ({"window": 1.5}, ValueError, "window must be positive and whole"),
            ({"scale": float("nan")}, ValueError, "scale"),
            ({"causal": False, "window": 3}, ValueError, "belong to the causal"),
            ({"causal": False, "prefix_lens": torch.tensor([1])}, ValueError, "belong"),
            ({"cu_seqlens_q": None}, ValueError, "cu_seqlens_q or q_seqinfo"),
            ({"cu_seqlens_k": None}, ValueError, "cu_seqlens_k or k_seqinfo"),
            ({"cu_seqlens_k": torch.tensor([0, 3, 6])}, AssertionError, "segment count")):
        args = {"cu_seqlens_q": c, "cu_seqlens_k": c, "q_seqinfo": None, "k_seqinfo": None,
                "causal": True, "window": None, "prefix_lens": None, "softcap": None,
                "scale": None, **kw}
        with pytest.raises(error, match=text):
            masked._check_options(64, **args)


def test_lengths_on_the_host():
    from varlenabsorbflashattn_amd import masked
    for bad in (torch.zeros(3), torch.zeros(3, dtype=torch.bool)):
        with pytest.raises(AssertionError, match="must be integers"):
            masked._host(bad, "prefix_lens")
    assert masked._host(torch.arange(8)[::2], "x").is_contiguous()
    a = torch.tensor([0, 3], dtype=torch.int32)
    key = _lib.ops().cu_key
    assert key(a) == key(a.clone()) != key(a.long()) and key(a) != key(a + 1)


def test_oracle_against_autograd():
    g = torch.Generator().manual_seed(0)
    H, Hk, D, ql, kl = 4, 2, 8, [5, 9], [5, 12]
    cq, ck = cu(ql), cu(kl)

    def rnd(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)
    q, k, v, do = rnd(14, H, D), rnd(17, Hk, D), rnd(17, Hk, D), rnd(14, H, D)
    slopes, cap, window, prefix = [0.5, 0.25, 0.1, 0.0], 2.0, 4, [2, 0]
    ref = om.attention(*(t.numpy() for t in (q, k, v, do)), cq, ck, 0.7, window=window,
                       prefix=prefix, softcap=cap, slopes=slopes)
    x = [t.requires_grad_(True) for t in (q, k, v)]
    outs = []
    for s in range(2):
        for h in range(H):
            qh, kh, vh = x[0][cq[s]:cq[s + 1], h], x[1][ck[s]:ck[s + 1], h // 2], \
                x[2][ck[s]:ck[s + 1], h // 2]
            z = cap * torch.tanh(0.7 * qh @ kh.T / cap)
            p = torch.arange(ql[s])[:, None] + kl[s] - ql[s]
            j = torch.arange(kl[s])
            z = z - slopes[h] * (p - j).abs().double()
            see = ((j <= p) & (j > p - window)) | (j < prefix[s])
            outs.append((torch.softmax(z.masked_fill(~see, -math.inf), 1) @ vh, s, h))
    loss = sum((o * do[cq[s]:cq[s + 1], h]).sum() for o, s, h in outs)
    for o, s, h in outs:
        np.testing.assert_allclose(ref["o"][0][cq[s]:cq[s + 1], h], o.detach().numpy(), atol=1e-12)
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(loss, x)):
        np.testing.assert_allclose(ref[name][0], got.numpy(), atol=1e-12)


def test_oracle_against_differences():
    g = np.random.default_rng(1)
    q, k, v, do = (g.standard_normal(s) for s in ((6, 2, 4), (7, 1, 4), (7, 1, 4), (6, 2, 4)))
    args = (np.array([0, 6]), np.array([0, 7]), -0.4)
    kw = {"softcap": 1.5, "slopes": [0.3, 0.1], "prefix": [3], "window": 2}
    ref = om.attention(q, k, v, do, *args, **kw)
    for name, i in (("dq", 0), ("dk", 1), ("dv", 2)):
        at, step = (2, 0, 1), 1e-6
        f = []
        for sign in (1, -1):
            x = [t.copy() for t in (q, k, v)]
            x[i][at] += sign * step
            f.append((om.attention(*x, None, *args, **kw)["o"][0] * do).sum())
        assert abs((f[0] - f[1]) / (2 * step) - ref[name][0][at]) < 1e-7


def test_oracle_rows_without_keys():
    g = np.random.default_rng(2)
    q, k, do = (g.standard_normal(s) for s in ((5, 1, 4), (2, 1, 4), (5, 1, 4)))
    ref = om.attention(q, k, k, do, np.array([0, 5]), np.array([0, 2]), 1.0, u=0.01)
    for n in ("o", "dq"):
        assert not ref[n][0][:3].any() and ref[n][0][3:].any()
        assert not ref[n][1][:3].any()


def test_expanded_slopes_are_refused():
    with pytest.raises(ValueError, match="alibi_slopes must be contiguous"):
        _call(alibi_slopes=torch.ones(1).expand(4))


def test_tangents_and_traces_are_refused():
    """Derivatives and traces that would lose the call without a word."""
    import torch.autograd.forward_ad as fw
    q, k = torch.zeros(6, 4, 64, dtype=torch.bfloat16), torch.zeros(6, 2, 64, dtype=torch.bfloat16)
    c, slopes = torch.tensor([0, 6], dtype=torch.int32), torch.ones(4)
    args = [q, k, k.clone(), slopes]

    def call(q, k, v, slopes):
        return packed_masked_attn(q, k, v, cu_seqlens_q=c, cu_seqlens_k=c, alibi_slopes=slopes)
    for at in range(4):
        for grad in (True, False):
            with fw.dual_level(), torch.set_grad_enabled(grad):
                x = [fw.make_dual(t, torch.ones_like(t)) if i == at else t
                     for i, t in enumerate(args)]
                with pytest.raises(ValueError, match="no forward-mode derivative"):
                    call(*x)
                x = [fw.unpack_dual(t).primal for t in x]
                with pytest.raises(AssertionError, match="requires GPU tensors"):
                    call(*x)
    with pytest.raises(ValueError, match="cannot be traced"):
        torch.jit.trace(call, tuple(args))
    with pytest.raises(AssertionError, match="requires GPU tensors"):
        call(*args)


def test_missing_pointers_are_refused_by_the_c_abi():
    L = _lib.lib()
    p = _lib.plan_masked(cu([4]), cu([4]), 4, 2, 64)
    ws = max(L.vafa_masked_fwd_workspace(p.info, 2, 64), L.vafa_masked_bwd_workspace(p.info, 2, 64))
    x = 1 << 20
    f = [x, x, x, x, x, x, x, p.info, 2, 64, _lib.DT_BF16, 0.1, 0.0, 0, None, x, ws, None]
    b = [x] * 11 + [p.info, 2, 64, _lib.DT_BF16, 0.1, 0.0, 0, None, x, ws, None]
    for call, args, required in ((L.vafa_masked_fwd, f, (0, 1, 2, 3, 6)),
                                 (L.vafa_masked_bwd, b, range(11))):
        for at in required:
            rc = call(*[None if i == at else y for i, y in enumerate(args)])
            assert rc == _lib.VAFA_ERR_VALUE, (call, at)
            assert at == 4 or "NULL" in _lib.last_error()


def test_prefix_lens_of_another_shape_are_refused_behind_a_cached_plan():
    from varlenabsorbflashattn_amd import masked
    q, k, c = torch.zeros(9, 2, 64), torch.zeros(9, 1, 64), cu([4, 5])
    c = torch.from_numpy(c)

    def plan(prefix):
        return masked._plan_of(q, k, c, c, True, 0, prefix)
    want = plan(torch.tensor([1, 3]))
    for bad in (torch.tensor([[1, 3]]), torch.tensor([[1], [3]]), torch.tensor([1, 3, 0])):
        with pytest.raises(AssertionError, match=r"prefix_lens must be \[2\]"):
            plan(bad)
    assert plan(torch.tensor([1, 3], dtype=torch.int32)) is want


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_bounds_tell_how_many_bits_of_o_delta_takes(dt):
    """Rows that few keys carry (steep distance biases): delta from o as the type holds it is
    outside the bounds, delta from eight more bits inside, each beside exact arithmetic."""
    u, a = {torch.bfloat16: (2.0 ** -8, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25)}[dt]
    g = torch.Generator().manual_seed(3)
    n, H, D = 60, 2, 64
    q, k, v, do = (torch.randn(n, H, D, generator=g).to(dt).double().numpy() for _ in range(4))
    at, slopes = np.array([0, n]), [4.0, 7.0]
    ref = om.attention(q, k, v, do, at, at, D ** -0.5, slopes=slopes, u=u, a=a)

    def gradients(bits):
        m, e = np.frexp(ref["o"][0])
        o = np.ldexp(np.round(m * 2.0 ** bits) / 2.0 ** bits, e)
        dq, dk = np.zeros_like(q), np.zeros_like(k)
        for h in range(H):
            P, _, _ = om._head(q[:, h], k[:, h], D ** -0.5, True, None, 0, None, slopes[h])
            dS = P * (do[:, h] @ v[:, h].T - (do[:, h] * o[:, h]).sum(1, keepdims=True)) * D ** -0.5
            dq[:, h], dk[:, h] = dS @ k[:, h], dS.T @ q[:, h]
        return dq, dk
    digits = 8 if dt == torch.bfloat16 else 11
    for bits, inside in ((digits, False), (digits + 8, True)):
        for name, x in zip(("dq", "dk"), gradients(bits)):
            val, bound = ref[name]
            assert bool((np.abs(x - val) <= bound).all()) == inside, (bits, name)
