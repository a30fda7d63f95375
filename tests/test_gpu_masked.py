"""Packed attention under a mask on the GPU against the 64-bit oracle, whose bounds count
the roundings element by element (oracle/masked.py)."""
import math

import numpy as np
import pytest
import torch

from oracle import masked as om
from varlenabsorbflashattn_amd import (packed_masked_attn, packed_varlen_attn, paged_decode_attn,
                                       paged_kv_append, set_validate_cu_seqlens)
from varlenabsorbflashattn_amd.workloads import cu_from_lens

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
A = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
BF, HF = torch.bfloat16, torch.float16


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def within(name, out, ref, bound):
    o = f64(out)
    assert o.shape == ref.shape and np.isfinite(o).all(), name
    d = np.abs(o - ref)
    worst = float((d / np.maximum(bound, 1e-300)).max()) if d.size else 0.0
    print(f"  {name:3s} max {d.max() if d.size else 0.0:.3e}, {worst:.2f} of the bound", flush=True)
    assert (d <= bound).all(), f"{name}: {worst} times the bound"


def inputs(case, ql, kl, H, Hk, D, dt, device, big=1.0):
    g = torch.Generator(device=device).manual_seed(case)

    def rnd(*s):
        return torch.randn(*s, generator=g, device=device)
    q = (big * rnd(sum(ql), H, D)).to(dt)
    return q, rnd(sum(kl), Hk, D).to(dt), rnd(sum(kl), Hk, D).to(dt), rnd(sum(ql), H, D).to(dt)


def step(q, k, v, do, ql, kl, **kw):
    """(o, dq, dk, dv) of one forward and backward."""
    x = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = packed_masked_attn(*x, cu_seqlens_q=cu_from_lens(ql), cu_seqlens_k=cu_from_lens(kl), **kw)
    return (o.detach(), *torch.autograd.grad(o, x, do))


def compare(got, q, k, v, do, ql, kl, *, scale=None, causal=True, window=None, prefix_lens=None,
            softcap=None, alibi_slopes=None):
    ref = om.attention(f64(q), f64(k), f64(v), f64(do), np.cumsum([0] + ql), np.cumsum([0] + kl),
                       scale if scale is not None else 1 / math.sqrt(q.shape[-1]), causal, window,
                       prefix_lens, softcap, f64(alibi_slopes), U[q.dtype], A[q.dtype])
    for (n, (val, bound)), out in zip(ref.items(), got):
        within(n, out, val, bound)


CASES = [
    # q lens, k lens (None: the same), H, Hk, D, dtype, options
    ([1], None, 1, 1, 64, BF, {}),
    ([5, 0, 300, 129, 1], None, 4, 2, 64, BF, {}),
    ([64, 63, 65, 128, 127, 257], None, 4, 4, 128, HF, {}),
    ([33, 200], None, 6, 1, 256, BF, {}),
    ([5, 40, 7, 3], [1, 900, 0, 3], 4, 4, 128, BF, {}),                 # rows without keys
    ([17, 500], [1000, 700], 8, 2, 128, BF, {"window": 50}),
    ([300, 33, 1], [300, 500, 2000], 4, 2, 256, HF, {"window": 64, "prefix_lens": [100, 500, 3]}),
    ([260, 10, 140], [300, 10, 140], 3, 3, 64, BF, {"prefix_lens": [300, 0, 77]}),
    ([130, 1, 40], [70, 900, 40], 4, 2, 128, HF, {"causal": False}),
    ([200, 31], None, 10, 2, 128, BF, {"softcap": 5.0}),
    ([200, 31], None, 4, 2, 256, BF, {"softcap": 30.0, "window": 100}),
    ([200, 31], None, 5, 1, 64, HF, {"softcap": 1.0}),
    ([150, 77], [150, 200], 12, 12, 64, BF, {"alibi": True}),
    ([150, 77], [150, 200], 3, 1, 128, HF, {"alibi": True, "prefix_lens": [40, 200]}),
    ([150, 77], [150, 200], 4, 4, 256, BF, {"alibi": True, "softcap": 20.0, "window": 33}),
    ([90, 20], None, 4, 2, 128, BF, {"alibi": True, "softcap": 20.0, "causal": False}),
    ([90, 20], None, 4, 2, 64, BF, {"scale": -0.3}),
    ([90, 20], None, 2, 2, 128, HF, {"scale": -0.3, "window": 7}),
    ([90, 20], None, 2, 1, 128, BF, {"scale": -0.3, "softcap": 2.0}),
    ([90, 20], None, 2, 1, 64, BF, {"scale": 0.0}),
    ([70, 9], None, 2, 1, 64, BF, {"window": 1}),                       # itself alone
    ([3, 1], [6000, 2500], 2, 1, 64, BF, {}),                           # split keys
    ([40, 16], [5000, 3000], 4, 1, 128, BF, {"window": 1500, "prefix_lens": [700, 0]}),
    ([100], [4000], 1, 1, 256, HF, {"softcap": 10.0, "alibi": True}),
    ([1] * 40, [1] * 40, 2, 2, 64, BF, {}),
    ([600, 700], None, 16, 8, 128, BF, {}),
    # head sets of 4, 8, 16 and 32 rows, two sets a key head, and a divided dK/dV pass
    ([50, 301], None, 24, 2, 64, BF, {"alibi": True}),
    ([50, 31], [200, 31], 8, 1, 128, HF, {"alibi": True, "window": 40}),
    ([9, 31], [9, 70], 16, 1, 64, BF, {"alibi": True, "softcap": 8.0}),
    ([1, 0, 37], None, 64, 1, 256, BF, {"alibi": True, "prefix_lens": [1, 0, 5]}),
    ([1500, 9], None, 16, 2, 64, BF, {}),
    ([900], None, 8, 1, 256, HF, {"softcap": 9.0}),
]


def options(kw, H, device):
    kw = dict(kw)
    if kw.pop("alibi", False):
        kw["alibi_slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)],
                                          device=device)
    if "prefix_lens" in kw:
        kw["prefix_lens"] = torch.tensor(kw["prefix_lens"], dtype=torch.int32)
    return kw


@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward_and_backward(device, case):
    ql, kl, H, Hk, D, dt, opts = CASES[case]
    kl = kl or ql
    print(f"[masked] q={ql[:6]} k={kl[:6]} H={H}/{Hk} D={D} {dt} {opts}", flush=True)
    x = inputs(case, ql, kl, H, Hk, D, dt, device)
    kw = options(opts, H, device)
    got = step(*x, ql, kl, **kw)
    torch.cuda.synchronize()
    if "prefix_lens" in kw:
        kw["prefix_lens"] = kw["prefix_lens"].numpy()
    compare(got, *x, ql, kl, **kw)


def test_gradients_against_differences(device):
    """The gradients of the calls themselves: f(x + e) - f(x - e) in 64 bits from the
    oracle moves as the GPU's gradients say."""
    ql, kl, H, Hk, D = [20], [23], 4, 2, 64
    print("[masked differences]", flush=True)
    x = inputs(50, ql, kl, H, Hk, D, HF, device)
    kw = {"softcap": 3.0, "window": 9, "prefix_lens": torch.tensor([4])}
    got = step(*x, ql, kl, **kw)
    h = [f64(t) for t in x]
    g = np.random.default_rng(0)
    for i, name in enumerate(("dq", "dk", "dv")):
        e = g.standard_normal(h[i].shape)
        f = []
        for sign in (1, -1):
            y = list(h[:3])
            y[i] = y[i] + sign * 1e-5 * e
            o = om.attention(*y, None, [0, 20], [0, 23], 0.125, window=9, prefix=[4], softcap=3.0)
            f.append((o["o"][0] * h[3]).sum())
        slope, along = (f[0] - f[1]) / 2e-5, (f64(got[1 + i]) * e).sum()
        # some 1e3 values with independent errors of a few 2^-11 of their size
        size = np.linalg.norm(f64(got[1 + i]) * e)
        print(f"  {name}: {along:.5f} against {slope:.5f}, norm {size:.3f}", flush=True)
        assert abs(along - slope) <= 8 * 2.0 ** -11 * size


def test_large_scores(device):
    """One-hot rows: scores in the hundreds, where every other probability underflows."""
    ql = [130, 40]
    print("[masked large]", flush=True)
    q, k, v, do = inputs(51, ql, ql, 4, 2, 64, BF, device, big=40.0)
    with torch.no_grad():
        o = packed_masked_attn(q, k, v, cu_seqlens_q=cu_from_lens(ql),
                               cu_seqlens_k=cu_from_lens(ql), scale=1.0)
    ref = om.attention(f64(q), f64(k), f64(v), None, np.cumsum([0] + ql), np.cumsum([0] + ql), 1.0,
                       u=U[BF])
    # scores of up to 2000 summed in fp32 over 64 products: P off by up to 2^-7
    val, bound = ref["o"]
    within("o", o, val, bound + 2.0 ** -7 * np.abs(f64(v)).max())


def test_not_causal_equals_packed_varlen(device):
    """Without the causal mask it is packed_varlen_attn, within both operators' roundings;
    shapes, layouts and lengths given as that operator takes them."""
    ql, kl = [40, 7], [300, 64]
    print("[masked varlen]", flush=True)
    q, k, v, do = inputs(52, ql, kl, 4, 4, 64, BF, device)
    info = {"q_seqinfo": torch.tensor(ql, device=device), "k_seqinfo": torch.tensor(kl, device=device)}
    a = packed_masked_attn(q[None], k[None], v[None], causal=False, **info)
    b = packed_varlen_attn(q[None], k[None], v[None], **info)
    assert a.shape == b.shape == (1, 47, 4, 64)
    ref = om.attention(f64(q), f64(k), f64(v), None, np.cumsum([0] + ql), np.cumsum([0] + kl), 0.125,
                       False, u=U[BF])["o"]
    within("o", a[0], *ref)
    within("o", b[0], *ref)
    # parts of a joint projection, and unaligned rows
    qkv = torch.randn(47, 12, 64, device=device).to(BF)
    views = qkv[:, :4], qkv[:, 4:8], qkv[:, 8:]
    kw = {"cu_seqlens_q": cu_from_lens(ql).to(device), "cu_seqlens_k": cu_from_lens(ql).to(device)}
    want = packed_masked_attn(*(t.contiguous() for t in views), **kw)
    assert torch.equal(packed_masked_attn(*views, **kw), want)
    flat = torch.zeros(47 * 4 * 64 + 1, device=device, dtype=BF)
    flat[1:] = views[0].flatten()
    assert torch.equal(packed_masked_attn(flat[1:].view(47, 4, 64), *views[1:], **kw), want)


def test_results_repeat(device):
    """The same bits from call to call, on another stream, and through calls of other
    lengths in between."""
    ql, kl = [500, 3, 130], [700, 3000, 130]
    print("[masked repeat]", flush=True)
    x = inputs(53, ql, kl, 8, 2, 128, BF, device)
    first = step(*x, ql, kl, window=600)
    step(*(t[:200] for t in x), [200], [200])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*x, ql, kl, window=600)
    again = step(*x, ql, kl, window=600)
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_rows_behind_the_last_segment(device):
    """With validation off, lengths may cover fewer rows than there are: zeros there."""
    print("[masked rest]", flush=True)
    ql = [30, 20]
    q, k, v, do = inputs(54, [70], [70], 2, 1, 64, BF, device)
    bad = torch.tensor(float("nan"), device=device).to(BF)
    q[50:], k[50:], v[50:], do[50:] = bad, bad, bad, bad
    set_validate_cu_seqlens(False)
    try:
        got = step(q, k, v, do, ql, ql)
    finally:
        set_validate_cu_seqlens(True)
    compare([t[:50] for t in got], q[:50], k[:50], v[:50], do[:50], ql, ql)
    assert not any(t[50:].any() for t in got)
    with pytest.raises(ValueError, match="must equal total tokens"):
        step(q, k, v, do, ql, ql)


def test_empty_calls(device):
    print("[masked empty]", flush=True)
    q = torch.zeros(0, 2, 64, device=device, dtype=BF, requires_grad=True)
    k = torch.ones(5, 1, 64, device=device, dtype=BF, requires_grad=True)
    o = packed_masked_attn(q, k, k, cu_seqlens_q=torch.tensor([0, 0]),
                           cu_seqlens_k=torch.tensor([0, 5]))
    o.sum().backward()
    assert o.shape == q.shape and not k.grad.any()
    q = torch.ones(4, 2, 64, device=device, dtype=BF, requires_grad=True)
    k = torch.zeros(0, 1, 64, device=device, dtype=BF, requires_grad=True)
    o = packed_masked_attn(q, k, k, cu_seqlens_q=torch.tensor([0, 4]),
                           cu_seqlens_k=torch.tensor([0, 0]))
    o.sum().backward()
    assert not o.any() and not q.grad.any() and k.grad.shape == k.shape


def test_training_step_under_graph_capture(device):
    """Forward and backward of two lengths in two graphs, replayed alternately with new
    values; eager work on tensors of its own in between."""
    print("[masked graph]", flush=True)
    g = torch.Generator(device=device).manual_seed(55)
    shapes = [([200, 7, 64], 4, 2, 64, {"softcap": 8.0}), ([90, 300], 4, 1, 128, {"window": 70})]
    state = []
    for ql, H, Hk, D, kw in shapes:
        x = [torch.zeros(sum(ql), n, D, device=device, dtype=BF) for n in (H, Hk, Hk, H)]
        state.append((x, ql, kw))
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g, device=device))
    graphs = []
    for x, ql, kw in state:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                step(*x, ql, ql, **kw)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*x, ql, ql, **kw)
        graphs.append((graph, out))
    for i in range(6):
        (x, ql, kw), (graph, out) = state[i % 2], graphs[i % 2]
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g, device=device))
        want = step(*(t.clone() for t in x), ql, ql, **kw)
        torch.cuda.synchronize()
        for t in out:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("opts", [{}, {"softcap": 10.0, "window": 40}, {"alibi": True}])
def test_decode_after_append_matches_the_packed_pass(device, opts):
    """A prompt through the packed attention and into the cache, then tokens one at a time:
    the last rows of the packed pass over the whole sequences, within both bounds."""
    print(f"[masked + paged] {opts}", flush=True)
    H, Hk, D, page, prompt, new = 8, 2, 128, 16, [37, 100, 1], 4
    kw = options(opts, H, device)
    total = [n + new for n in prompt]
    cu, cu_p = cu_from_lens(total), cu_from_lens(prompt)
    g = torch.Generator(device=device).manual_seed(56)
    qkv = torch.randn(sum(total), H + 2 * Hk, D, generator=g, device=device).to(BF)
    inv = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().to(device)
    pages = [-(-n // page) for n in total]
    table = torch.full((3, max(pages)), -1, dtype=torch.int32)
    order, at = torch.randperm(sum(pages)).int(), 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    table = table.to(device)

    def caches():
        return [torch.full((sum(pages), page, Hk, D), float("nan"), device=device).to(BF)
                for _ in range(2)]

    def parts(x):
        return x[:, H:H + Hk], x[:, H + Hk:]
    # the whole sequences at once: rotated q and k for the packed pass
    zero = torch.zeros(3, dtype=torch.int32, device=device)
    kc, vc = caches()
    q = paged_kv_append(*parts(qkv), kc, vc, table, zero, cu_seqlens=cu.to(device), q=qkv[:, :H],
                        inv_freq=inv)
    rows = torch.cat([table[b].long()[torch.arange(n, device=device) // page] * page
                      + torch.arange(n, device=device) % page for b, n in enumerate(total)])
    k, v = (c.flatten(0, 1)[rows] for c in (kc, vc))
    assert torch.equal(v, qkv[:, H + Hk:])
    o = packed_masked_attn(q, k, v, cu_seqlens_q=cu, cu_seqlens_k=cu, **kw)
    val, bound = om.attention(f64(q), f64(k), f64(v), None, cu.numpy(), cu.numpy(), D ** -0.5,
                              window=kw.get("window"), softcap=kw.get("softcap"),
                              slopes=f64(kw.get("alibi_slopes")), u=U[BF])["o"]
    within("o", o, val, bound)
    # prompt, then step by step
    kc2, vc2 = caches()
    first = torch.cat([torch.arange(cu[b], cu[b] + n) for b, n in enumerate(prompt)]).to(device)
    paged_kv_append(*parts(qkv[first]), kc2, vc2, table, zero, cu_seqlens=cu_p.to(device),
                    inv_freq=inv)
    lens = torch.tensor(prompt, dtype=torch.int32, device=device)
    for t in range(new):
        at = (cu[:-1] + torch.tensor(prompt) + t).to(device)
        x = qkv[at]
        qs = paged_kv_append(*parts(x), kc2, vc2, table, lens, q=x[:, :H], inv_freq=inv)
        lens += 1
        assert torch.equal(qs, q[at])
        out = paged_decode_attn(qs, kc2, vc2, table, lens, **kw)
        i = at.cpu().numpy()
        within("o", out, val[i], bound[i])
    same = torch.equal(torch.nan_to_num(kc), torch.nan_to_num(kc2))
    assert same and torch.equal(torch.nan_to_num(vc), torch.nan_to_num(vc2))


def test_shared_and_expanded_keys(device):
    """Keys that one tensor gives to two segments, values expanded over the key heads: the
    copies' gradients add up in the leaf."""
    print("[masked expanded]", flush=True)
    n, H, Hk, D = 40, 4, 2, 64
    q, k, v, do = inputs(57, [2 * n], [n], H, Hk, D, HF, device)
    x = [t.detach().requires_grad_(True) for t in (q, k, v[:, :1])]
    kk, vv = torch.cat([x[1], x[1]]), x[2].expand(n, Hk, D).repeat(2, 1, 1)
    cu = cu_from_lens([n, n])
    o = packed_masked_attn(x[0], kk, vv, cu_seqlens_q=cu, cu_seqlens_k=cu)
    dq, dk, dv = torch.autograd.grad(o, x, do)
    ref = om.attention(f64(q), f64(kk), f64(vv), f64(do), [0, n, 2 * n], [0, n, 2 * n], D ** -0.5,
                       u=U[HF], a=A[HF])
    within("dq", dq, *ref["dq"])
    val, bound = (np.add(x[:n], x[n:]) for x in ref["dk"])
    u = U[HF]  # torch adds the two in fp16 again
    within("dk", dk, val, bound + u * np.abs(val) + A[HF])
    val, bound = (x.reshape(2, n, Hk, D).sum((0, 2))[:, None] for x in ref["dv"])
    mag = np.abs(ref["dv"][0]).reshape(2, n, Hk, D).sum((0, 2))[:, None]
    within("dv", dv, val, bound + 3 * (u * mag + A[HF]))


def test_needs_grad_of_some(device):
    """Gradients of k and v alone, of q alone, and a second derivative refused."""
    print("[masked some]", flush=True)
    ql = [70]
    x = inputs(58, ql, ql, 4, 2, 64, BF, device)
    want = step(*x, ql, ql)
    cu = cu_from_lens(ql)
    for need in ((0,), (1, 2), (2,)):
        y = [t.detach().requires_grad_(i in need) for i, t in enumerate(x[:3])]
        o = packed_masked_attn(*y, cu_seqlens_q=cu, cu_seqlens_k=cu)
        got = torch.autograd.grad(o, [y[i] for i in need], x[3])
        for i, t in zip(need, got):
            assert torch.equal(t, want[1 + i])
    y = [t.detach().requires_grad_(True) for t in x[:3]]
    o = packed_masked_attn(*y, cu_seqlens_q=cu, cu_seqlens_k=cu)
    g, = torch.autograd.grad(o, y[:1], x[3], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), y[1])


def test_two_threads(device):
    """Calls of different lengths from two threads, each on a stream of its own."""
    import threading
    print("[masked threads]", flush=True)
    cases = []
    for i, (ql, kw) in enumerate((([200, 50], {"window": 60}), ([90, 300], {"softcap": 4.0}))):
        x = inputs(59 + i, ql, ql, 4, 2, 64, BF, device)
        cases.append((x, ql, kw, step(*x, ql, ql, **kw)))
    torch.cuda.synchronize()
    errors = []

    def work(x, ql, kw, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = step(*x, ql, ql, **kw)
                torch.cuda.current_stream().synchronize()
            for a, b in zip(got, want):
                assert torch.equal(a, b)
        except BaseException as e:
            errors.append(e)
    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_past_4_gib(device):
    """Tensors of more than 4 GiB: the last segment, a copy of the first, gives its bits."""
    n, seg, H, D = 2200, 512, 16, 128
    print(f"[masked far] {n} x {seg} tokens, {n * seg * H * D * 2 / 2 ** 30:.1f} GiB each",
          flush=True)
    g = torch.Generator(device=device).manual_seed(60)
    x = []
    for _ in range(4):
        t = torch.empty(n * seg, H, D, device=device, dtype=BF)
        t.view(n, seg * H * D).copy_(torch.randn(1, seg * H * D, generator=g, device=device))
        x.append(t)
    lens = [seg] * n
    got = step(*x, lens, lens, window=100)
    near = step(*(t[:seg] for t in x), [seg], [seg], window=100)
    for far, one in zip(got, near):
        assert torch.equal(far[-seg:], one) and torch.equal(far[:seg], one)
    small = [t[:seg, :2] for t in x]
    compare([t[:, :2] for t in near], *small, [seg], [seg], window=100)


@pytest.mark.parametrize("ql,kl,H,Hk,D,dt", [([200, 7, 33], None, 4, 2, 64, BF),
                                             ([130, 1, 61], None, 6, 1, 128, HF),
                                             ([100], [4000], 2, 1, 128, BF),
                                             ([90, 21], [90, 3500], 2, 2, 256, HF)])
def test_gradients_of_rows_that_few_keys_carry(device, ql, kl, H, Hk, D, dt):
    """Steep distance biases: dP - delta is far below either, so that O's rounding in delta
    alone would put dQ and dK 3 to 8 u off.  What stays is the rounding of dS for the
    product and that of the result, independent and of at most u / sqrt(3) each in the mean:
    0.82 u of the norm."""
    print(f"[masked steep] {ql} {kl} {H}/{Hk} x {D} {dt}", flush=True)
    kl = kl or ql
    x = inputs(61, ql, kl, H, Hk, D, dt, device)
    slopes = torch.linspace(4.0, 7.0, H, device=device)
    got = step(*x, ql, kl, alibi_slopes=slopes)
    ref = om.attention(*(f64(t) for t in x), np.cumsum([0] + ql), np.cumsum([0] + kl), D ** -0.5,
                       slopes=f64(slopes), u=U[dt], a=A[dt])
    for name, out in zip(("o", "dq", "dk", "dv"), got):
        val = ref[name][0]
        off = np.linalg.norm(f64(out) - val) / np.linalg.norm(val)
        print(f"  {name:3s} {off / U[dt]:.2f} u", flush=True)
        assert off < U[dt], (name, off)


def test_many_tiny_segments(device):
    """20000 segments of one token: each gets its own value, dQ and dK are zeros and dV the sum
    over the heads that share it (small whole numbers: exact)."""
    print("[masked tiny]", flush=True)
    n, H, Hk, D = 20000, 6, 3, 64
    g = torch.Generator(device=device).manual_seed(62)
    q, k, v = (torch.randn(n, h, D, generator=g, device=device).to(BF).requires_grad_(True)
               for h in (H, Hk, Hk))
    do = torch.randint(-8, 9, (n, H, D), generator=g, device=device).to(BF)
    cu = torch.arange(n + 1)
    o = packed_masked_attn(q, k, v, cu_seqlens_q=cu, cu_seqlens_k=cu, window=3)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    assert torch.equal(o, v.repeat_interleave(H // Hk, dim=1))
    assert torch.equal(dv, do.view(n, Hk, H // Hk, D).sum(2))
    # dP - delta: two fp32 sums of the same 64 products, each off by at most 66 roundings
    off = 2 * 66 * 2.0 ** -24 * (do.float() * o.float()).abs().sum(-1).max() * D ** -0.5 * 1.01
    assert dq.abs().max() <= off * k.abs().max()
    assert dk.abs().max() <= off * q.abs().max() * (H // Hk)


@pytest.mark.parametrize("H,Hk,D", [(4096, 1, 64), (4096, 4096, 64), (96, 32, 256)])
def test_most_heads(device, H, Hk, D):
    print(f"[masked heads] {H}/{Hk} x {D}", flush=True)
    ql, kl = [5, 2], [5, 40]
    x = inputs(63, ql, kl, H, Hk, D, HF, device)
    compare(step(*x, ql, kl), *x, ql, kl)


@pytest.mark.parametrize("seed", range(16))
def test_random_masks(device, seed):
    rng = np.random.RandomState(100 + seed)
    D, dt = (64, 128, 256)[seed % 3], (BF, HF)[seed % 2]
    Hk = int(rng.choice([1, 2, 3]))
    H = Hk * int(rng.choice([1, 2, 3, 4, 8]))
    n = int(rng.randint(1, 6))
    ql = [int(x) for x in rng.randint(0, 200, n)]
    kl = [int(x) for x in (rng.randint(0, 400, n) if rng.rand() < 0.5 else ql)]
    kw = {}
    if rng.rand() < 0.7:
        kw["window"] = int(rng.choice([1, 2, 31, 64, 65, 150]))
    if rng.rand() < 0.6:
        kw["prefix_lens"] = [int(rng.randint(0, k + 1)) for k in kl]
    if rng.rand() < 0.3:
        kw["softcap"] = float(rng.choice([2.0, 30.0]))
    if rng.rand() < 0.3:
        kw["alibi_slopes"] = torch.linspace(0.01, 0.5, H, device=device)
    print(f"[masked random {seed}] {ql} {kl} {H}/{Hk} x {D} {dt} {kw}", flush=True)
    if sum(ql) == 0 or sum(kl) == 0:
        ql, kl = ql + [3], kl + [4]
        if "prefix_lens" in kw:
            kw["prefix_lens"] = kw["prefix_lens"] + [1]
    x = inputs(200 + seed, ql, kl, H, Hk, D, dt, device)
    compare(step(*x, ql, kl, **kw), *x, ql, kl, **kw)


@pytest.mark.parametrize("D,dt,opts", [(64, BF, {}), (128, HF, {"softcap": 20.0}), (256, BF, {}),
                                       (128, BF, {"alibi": True}), (64, HF, {"softcap": 5.0})])
def test_unseen_keys_and_rows_without_keys_hold_anything(device, D, dt, opts):
    """NaN and infinities in keys that no query sees (in front of the window) and in queries
    and gradients of rows that see no key change nothing: zeros come out for them."""
    print(f"[masked unseen] {D} {dt} {opts}", flush=True)
    opts = dict(opts)
    H, Hk, w = 4, 2, 40
    ql, kl = [70, 100, 150], [300, 100, 90]  # 60 rows of the last segment see nothing
    x = inputs(64, ql, kl, H, Hk, D, dt, device)
    if opts.pop("alibi", False):
        opts["alibi_slopes"] = torch.linspace(0.1, 0.4, H, device=device)
    k_dead = slice(0, 300 - 70 - w + 1)
    q_dead = slice(170, 170 + 60)
    want, got = [t.clone() for t in x], [t.clone() for t in x]
    for i, s in ((0, q_dead), (3, q_dead), (1, k_dead), (2, k_dead)):
        want[i][s] = 0
        got[i][s] = float("nan") if i != 2 else float("inf")
    a, b = (step(*y, ql, kl, window=w, **opts) for y in (got, want))
    for name, s, t in zip(("o", "dq", "dk", "dv"), a, b):
        assert torch.isfinite(s).all(), name
        assert torch.equal(s, t), name
    assert not a[0][q_dead].any() and not a[1][q_dead].any()
    assert not a[2][k_dead].any() and not a[3][k_dead].any()


def test_second_derivatives_are_refused(device):
    """With create_graph a gradient is no constant: what would need a second derivative
    raises, also inside a sum with terms that have one."""
    print("[masked second]", flush=True)
    ql = [40, 9]
    x = inputs(65, ql, ql, 4, 2, 64, BF, device)
    want = step(*x, ql, ql)
    cu = cu_from_lens(ql)
    y = [t.detach().requires_grad_(True) for t in x[:3]]
    w = torch.ones(4, 1, device=device, dtype=BF, requires_grad=True)
    o = packed_masked_attn(*y, cu_seqlens_q=cu, cu_seqlens_k=cu)
    grads = torch.autograd.grad(o, y, x[3], create_graph=True)
    for a, b in zip(grads, want[1:]):
        assert a.requires_grad and torch.equal(a, b)
    refused = pytest.raises(RuntimeError, match="packed_masked_attn has no second derivative")
    for at in range(3):
        with refused:
            (o.float().sum() + grads[at].float().square().sum()).backward(retain_graph=True)
        for i in range(3):
            with refused:
                torch.autograd.grad(grads[at].sum(), y[i], allow_unused=True, retain_graph=True)
    # an upstream gradient that requires one; products of constants keep their derivatives
    do = x[3].detach().requires_grad_(True)
    o = packed_masked_attn(*y, cu_seqlens_q=cu, cu_seqlens_k=cu)
    g, = torch.autograd.grad(o, y[:1], do, create_graph=True)
    with refused:
        torch.autograd.grad(g.sum(), do, retain_graph=True)
    d, = torch.autograd.grad((g * w).sum(), w)
    assert torch.equal(d, torch.autograd.grad((want[1] * w).sum(), w)[0])
    # without create_graph, constants as before
    y = [t.detach().requires_grad_(True) for t in x[:3]]
    packed_masked_attn(*y, cu_seqlens_q=cu, cu_seqlens_k=cu).backward(x[3])
    assert not any(t.grad.requires_grad for t in y)


@pytest.mark.parametrize("ql,kl,H,Hk,D,dt", [([200, 7, 33], None, 4, 2, 64, BF),
                                             ([130, 1, 61], None, 6, 1, 128, HF),
                                             ([100], [4000], 2, 1, 128, BF),
                                             ([90, 21], [90, 3500], 2, 2, 256, HF)])
def test_elements_of_rows_that_few_keys_carry(device, ql, kl, H, Hk, D, dt):
    """Steep distance biases, element by element: the bounds there are below what delta from
    o in the type's own bits would give (tests/test_masked.py)."""
    print(f"[masked steep elements] {ql} {kl} {H}/{Hk} x {D} {dt}", flush=True)
    kl = kl or ql
    x = inputs(66, ql, kl, H, Hk, D, dt, device)
    slopes = torch.linspace(4.0, 7.0, H, device=device)
    compare(step(*x, ql, kl, alibi_slopes=slopes), *x, ql, kl, alibi_slopes=slopes)


def test_prompt_behind_a_cached_prefix(device):
    """Several new tokens behind what the cache holds: appended, the sequences' keys and
    values gathered from their pages, and the packed pass over more keys than queries.  Its
    rows are those of a pass over the whole sequences."""
    H, Hk, D, page, past, new = 4, 2, 64, 16, [70, 0, 33], [40, 25, 1]
    print(f"[masked prefix cache] {past} + {new}", flush=True)
    total = [a + b for a, b in zip(past, new)]
    g = torch.Generator(device=device).manual_seed(67)
    qkv = torch.randn(sum(total), H + 2 * Hk, D, generator=g, device=device).to(HF)
    pages = [-(-n // page) for n in total]
    table = torch.full((3, max(pages)), -1, dtype=torch.int32)
    order = torch.randperm(sum(pages), generator=torch.Generator().manual_seed(67)).int()
    for b, n in enumerate(pages):
        table[b, :n] = order[sum(pages[:b]):sum(pages[:b + 1])]
    page_table = table.to(device)
    # a joint allocation: keys and values of a page beside each other
    both = torch.full((sum(pages), 2, page, Hk, D), float("nan"), device=device).to(HF)
    k_cache, v_cache = both[:, 0], both[:, 1]
    inv = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().to(device)
    seq = torch.repeat_interleave(torch.arange(3), torch.tensor(total))
    pos = torch.cat([torch.arange(n) for n in total])
    old = (pos < torch.tensor(past)[seq]).to(device)
    lens = torch.zeros(3, dtype=torch.int32, device=device)
    qs = []
    for rows, n in ((old, past), (~old, new)):
        x = qkv[rows]
        qs.append(paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], k_cache, v_cache, page_table, lens,
                                  cu_seqlens=cu_from_lens(n).int().to(device), q=x[:, :H],
                                  inv_freq=inv))
        lens += torch.tensor(n, dtype=torch.int32, device=device)
    b, pos = seq.to(device), pos.to(device)
    at = page_table[b, pos // page].long()
    k, v = k_cache[at, pos % page], v_cache[at, pos % page]
    assert torch.equal(v, qkv[:, H + Hk:])
    kw = {"window": 50, "softcap": 20.0}
    o = packed_masked_attn(qs[1], k, v, cu_seqlens_q=cu_from_lens(new),
                           cu_seqlens_k=cu_from_lens(total), **kw)
    q = torch.empty_like(qkv[:, :H])
    q[old], q[~old] = qs
    val, bound = om.attention(f64(q), f64(k), f64(v), None, np.cumsum([0] + total),
                              np.cumsum([0] + total), D ** -0.5, u=U[HF], a=A[HF], **kw)["o"]
    keep = (~old).cpu().numpy()
    within("o", o, val[keep], bound[keep])


def test_saved_tensors_elsewhere(device):
    """Gradients with the saved tensors kept on the host, and recomputed by checkpointing."""
    from torch.utils.checkpoint import checkpoint
    print("[masked saved]", flush=True)
    ql = [90, 31]
    x = inputs(68, ql, ql, 4, 2, 128, BF, device)
    slopes = torch.linspace(0.1, 0.4, 4, device=device)
    kw = {"window": 40, "alibi_slopes": slopes}
    want = step(*x, ql, ql, **kw)

    def call(q, k, v):
        return packed_masked_attn(q, k, v, cu_seqlens_q=cu_from_lens(ql),
                                  cu_seqlens_k=cu_from_lens(ql), **kw)
    y = [t.detach().requires_grad_(True) for t in x[:3]]
    with torch.autograd.graph.save_on_cpu():
        o = call(*y)
    for a, b in zip((o, *torch.autograd.grad(o, y, x[3])), want):
        assert torch.equal(a, b)
    for reentrant in (False, True):
        y = [t.detach().requires_grad_(True) for t in x[:3]]
        o = checkpoint(call, *y, use_reentrant=reentrant)
        o.backward(x[3])
        for a, b in zip((o, *(t.grad for t in y)), want):
            assert torch.equal(a, b)
