"""Paged key-value cache on the GPU against the 64-bit oracle.

Bounds, element by element (u: half a step of the type relative to a value, 2^-8 bf16,
2^-11 fp16; a: half the smallest step of fp16, 2^-25; both apply to what is rounded):

* append: one rounding of the turned pair, u |y| + a, after fp32 sums of two products
  whose sine and cosine are off by a few fp32 steps: 2^-20 (|x1| + |x2|).  Keys that are
  not turned, values and untouched slots are equal.
* decode: probabilities are rounded for the product (u P each, fp16 also a) and their
  rounded values summed, so numerator and denominator are each off by u: 2 u sum P |v|
  + 2 a sum |v| / l; the scores' fp32 sums move P by less than 2^-12 at the sizes here;
  then the output's own rounding u |o| + a.
"""
import math

import numpy as np
import pytest
import torch

from oracle import paged as op
from varlenabsorbflashattn_amd import paged_decode_attn, paged_kv_append

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
A = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def f64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def within(name, out, ref, bound):
    o = f64(out)
    assert np.isfinite(o).all(), name
    d = np.abs(o - ref)
    worst = float((d / np.maximum(bound, 1e-300)).max()) if d.size else 0.0
    print(f"  {name}: max {d.max() if d.size else 0.0:.3e}, {worst:.2f} of the bound", flush=True)
    assert (d <= bound).all(), f"{name}: {worst} times the bound"


def close_decode(out, ref, mag, flat):
    u, a = U[out.dtype], A[out.dtype]
    within("out", out, ref, (2 * u + 2.0 ** -12) * mag + 2 * a * flat + u * np.abs(ref) + a)


def cache_pair(g, n_pages, page, Hk, D, dt, device, layout):
    """Two caches in one of the layouts a serving loop keeps."""
    def rnd(*s):
        return torch.randn(*s, generator=g, device=device).to(dt)
    if layout == "joint":
        both = rnd(n_pages, 2, page, Hk, D)
        return both[:, 0], both[:, 1]
    if layout == "heads":
        return (rnd(n_pages, Hk, page, D).transpose(1, 2) for _ in range(2))
    return rnd(n_pages, page, Hk, D), rnd(n_pages, page, Hk, D)


def pages_for(g, lens, page, spare=2, width=None):
    """A page table of distinct pages in random order, unused entries garbage."""
    need = [-(-n // page) for n in lens]
    N = sum(need) + spare
    order = torch.randperm(N, generator=torch.Generator().manual_seed(int(g.initial_seed()))).numpy()
    table = np.full((len(lens), width or max(max(need), 1)), 1 << 30, np.int64)
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    return torch.from_numpy(table.astype(np.int32)), N


APPEND = [
    # lens (None: one token each), past, H, Hk, D, page, rotated, interleaved, dtype, layout
    (None, [0, 1, 15, 16, 500], 4, 2, 64, 16, 64, False, torch.bfloat16, "plain"),
    (None, [7, 100000, 3], 8, 8, 128, 256, 128, False, torch.float16, "joint"),
    ([5, 0, 33, 1], [0, 9, 14, 31], 6, 3, 128, 16, 64, True, torch.bfloat16, "heads"),
    ([130, 64], [1, 0], 5, 1, 256, 64, 256, False, torch.float16, "plain"),
    ([3, 20], [2, 4], 2, 2, 64, 7, 20, True, torch.bfloat16, "plain"),   # odd pages and pairs
    ([3, 20], [2, 4], 2, 2, 80, 1, 40, False, torch.float16, "joint"),
    ([17, 2], [0, 0], 1, 1, 128, 32, 0, False, torch.bfloat16, "plain"),  # no rotation
    ([1] * 130, [i * 3 for i in range(130)], 2, 1, 64, 16, 32, False, torch.bfloat16, "plain"),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(device, case):
    lens, past, H, Hk, D, page, rot, inter, dt, layout = APPEND[case]
    print(f"[append] {APPEND[case]}", flush=True)
    g = torch.Generator(device=device).manual_seed(case + 1)
    new = [1] * len(past) if lens is None else lens
    T, extra = sum(new), 0 if lens is None else 5  # rows behind the last sequence
    qkv = torch.randn(T + extra, H + 2 * Hk, D, generator=g, device=device).to(dt)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    table, N = pages_for(g, [a + b for a, b in zip(new, past)], page)
    kc, vc = cache_pair(g, N, page, Hk, D, dt, device, layout)
    cu = None if lens is None else torch.tensor(np.cumsum([0] + new), dtype=torch.int32)
    inv = (10000.0 ** (-torch.arange(0, rot, 2) / rot)).float() if rot else None
    plens = torch.tensor(past, dtype=torch.int32)
    want = op.append(f64(k), f64(v), f64(kc), f64(vc), table.numpy(), past,
                     None if cu is None else cu.numpy(), f64(q), f64(inv), inter)
    versions = kc._version, vc._version
    out = paged_kv_append(k, v, kc, vc, table.to(device), plens.to(device),
                          cu_seqlens=None if cu is None else cu.to(device), q=q,
                          inv_freq=None if inv is None else inv.to(device), interleaved=inter)
    torch.cuda.synchronize()
    assert kc._version > versions[0] and vc._version > versions[1]
    u, a = U[dt], A[dt]
    for name, got, ref, mag in (("q", out, want[0], want[3]), ("k", kc, want[1], want[4])):
        within(name, got, ref, u * np.abs(ref) + a + 2.0 ** -20 * mag)
        rest = f64(got)[..., rot:]
        assert np.array_equal(rest, ref[..., rot:]), name
    assert np.array_equal(f64(vc), want[2])
    assert not out[T:].any()
    # without q, into a second pair of caches: the same bits
    k2, v2 = kc.clone(), vc.clone()
    assert paged_kv_append(k, v, k2, v2, table.to(device), plens.to(device),
                           cu_seqlens=None if cu is None else cu.to(device),
                           inv_freq=None if inv is None else inv.to(device),
                           interleaved=inter) is None
    assert torch.equal(k2, kc) and torch.equal(v2, vc)


def test_append_far_positions(device):
    """Angles of positions whose product with the frequency has no fraction left in
    32 bits; a table of one page holds them through a page as long."""
    print("[append far]", flush=True)
    D, pos = 64, [2 ** 24 + 1, 10 ** 8 + 7, 2 ** 31 - 2]
    g = torch.Generator(device=device).manual_seed(3)
    q = torch.randn(3, 2, D, generator=g, device=device).to(torch.float16)
    k = torch.randn(3, 1, D, generator=g, device=device).to(torch.float16)
    kc = torch.zeros(1, 16, 1, D, device=device, dtype=torch.float16)
    inv = (10000.0 ** (-torch.arange(0, D, 2) / D)).float()
    # one page of 16 tokens: the positions lie past it, so only q comes back
    out = paged_kv_append(k, k, kc, kc.clone(), torch.zeros(3, 1, dtype=torch.int32, device=device),
                          torch.tensor(pos, dtype=torch.int32, device=device), q=q,
                          inv_freq=inv.to(device))
    ref, mag = op.rotate(f64(q), np.array(pos), f64(inv), False)
    within("q", out, ref, U[q.dtype] * np.abs(ref) + A[q.dtype] + 2.0 ** -19 * mag)
    assert not kc.any()


def test_append_outside(device):
    """Bad pages, positions outside the table and negative lengths store nothing."""
    print("[append outside]", flush=True)
    dt, page, Hk, D = torch.bfloat16, 16, 2, 64
    g = torch.Generator(device=device).manual_seed(4)
    kc, vc = cache_pair(g, 3, page, Hk, D, dt, device, "plain")
    k = torch.randn(6, Hk, D, generator=g, device=device).to(dt)
    table = torch.tensor([[3, 0], [-1, 0], [1, 2 ** 31 - 1], [1, 2], [0, 1], [2, 0]],
                         dtype=torch.int32)
    lens = torch.tensor([0, 3, 16, 32, -1, 17], dtype=torch.int32)
    want = op.append(f64(k), f64(k), f64(kc), f64(vc), table.numpy(), lens.numpy(), None, None,
                     None, False)
    before = kc.clone()
    paged_kv_append(k, k, kc, vc, table.to(device), lens.to(device))
    assert np.array_equal(f64(kc), want[1]) and np.array_equal(f64(vc), want[2])
    assert int((kc != before).any(-1).any(-1).sum()) == 1  # the last token alone found a place


DECODE = [
    # lens, H, Hk, D, page, softcap, window, slopes, dtype, layout
    ([1, 2, 0, 17, 130, 500], 4, 1, 64, 16, None, None, False, torch.bfloat16, "plain"),
    ([127, 128, 129, 1], 8, 8, 128, 16, None, None, False, torch.float16, "joint"),
    ([1000, 31], 40, 2, 128, 7, None, None, True, torch.bfloat16, "heads"),  # 20 heads a key head
    ([700, 5, 64], 6, 2, 256, 64, 30.0, None, False, torch.float16, "plain"),
    ([900, 100, 1], 4, 4, 64, 1, 5.0, 100, True, torch.bfloat16, "plain"),
    ([300, 2000], 16, 1, 256, 256, 50.0, 128, False, torch.bfloat16, "joint"),
    ([40] * 70 + [300], 2, 2, 64, 16, None, None, False, torch.bfloat16, "plain"),
    ([5000], 3, 1, 128, 48, None, 1, False, torch.float16, "plain"),
    ([0, 0], 4, 2, 64, 16, None, None, False, torch.bfloat16, "plain"),
    ([20000, 3, 9000], 8, 4, 128, 32, None, None, False, torch.bfloat16, "plain"),
    ([6000], 64, 1, 256, 128, None, 4097, True, torch.float16, "heads"),
]


def decode_case(case, device, big=1.0):
    lens, H, Hk, D, page, cap, window, alibi, dt, layout = DECODE[case]
    g = torch.Generator(device=device).manual_seed(case + 11)
    table, N = pages_for(g, lens, page)
    kc, vc = cache_pair(g, N, page, Hk, D, dt, device, layout)
    # q as a part of a joint projection
    q = (big * torch.randn(len(lens), H + 3, D, generator=g, device=device)).to(dt)[:, :H]
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)]) if alibi else None
    kw = {"softcap": cap, "window": window}
    return lens, q, kc, vc, table, slopes, kw


@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode(device, case):
    print(f"[decode] {DECODE[case][1:]}", flush=True)
    lens, q, kc, vc, table, slopes, kw = decode_case(case, device)
    out = paged_decode_attn(q, kc, vc, table.to(device),
                            torch.tensor(lens, dtype=torch.int32, device=device),
                            alibi_slopes=None if slopes is None else slopes.to(device), **kw)
    ref = op.decode(f64(q), f64(kc), f64(vc), table.numpy(), lens, 1 / math.sqrt(q.shape[-1]),
                    slopes=f64(slopes), **kw)
    close_decode(out, *ref)


def test_decode_absent_keys(device):
    """What lies behind a length, in bad pages or in front of the window is not read as
    values: infinities and NaN there do not reach the result."""
    print("[decode absent]", flush=True)
    dt, page, Hk, D, H = torch.bfloat16, 16, 2, 64, 4
    g = torch.Generator(device=device).manual_seed(5)
    lens, window = [37, 90, 200, 5], 50
    table, N = pages_for(g, lens, page, width=13)
    table[1, 4] = N + 3
    table[2, 10], table[2, 11] = -7, 2 ** 31 - 1
    table[3, 0] = -1  # no page at all: zeros
    kc, vc = cache_pair(g, N, page, Hk, D, dt, device, "plain")
    seen = torch.zeros(N, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(max(0, n - window), n):
            at = op.place(table.numpy(), N, page, b, j)
            if at is not None:
                seen[at] = True
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")], device=device).to(dt)
    kb, vb = kc.clone(), vc.clone()
    hidden = (~seen).to(device)
    kb[hidden] = bad[torch.randint(3, kb[hidden].shape, generator=g, device=device)]
    vb[hidden] = bad[torch.randint(3, vb[hidden].shape, generator=g, device=device)]
    q = torch.randn(4, H, D, generator=g, device=device).to(dt)
    args = (table.to(device), torch.tensor(lens, dtype=torch.int32, device=device))
    out = paged_decode_attn(q, kb, vb, *args, window=window)
    ref = op.decode(f64(q), f64(kc), f64(vc), table.numpy(), lens, 1 / math.sqrt(D), window=window)
    close_decode(out, *ref)
    assert not out[3].any()
    # lengths past the table count as full, negative ones as none
    far = torch.tensor([2 ** 31 - 1, -4, 13 * page + 1, -2 ** 31], dtype=torch.int32)
    out = paged_decode_attn(q, kc, vc, table.to(device), far.to(device))
    ref = op.decode(f64(q), f64(kc), f64(vc), table.numpy(), far.tolist(), 1 / math.sqrt(D))
    close_decode(out, *ref)


def test_decode_large_scores(device):
    """Scores in the thousands (one-hot rows) and a negative scale."""
    print("[decode large]", flush=True)
    lens, q, kc, vc, table, slopes, kw = decode_case(0, device, big=30.0)
    args = (q, kc, vc, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device))
    for scale in (1.0, -0.05):
        out = paged_decode_attn(*args, scale=scale)
        ref, mag, flat = op.decode(f64(q), f64(kc), f64(vc), table.numpy(), lens, scale)
        # scores of up to 2000 in fp32: off by 64 products of 2^-24 of their size, so P by 2^-7
        u = U[q.dtype]
        within("out", out, ref, (2 * u + 2.0 ** -7) * mag + u * np.abs(ref))


def test_decode_after_append_matches_whole_sequence(device):
    """A prompt appended at once, then tokens one at a time, each attended: as they would
    be used together.  The result of every step is the oracle's on the cache's contents."""
    print("[append + decode]", flush=True)
    dt, H, Hk, D, page, steps = torch.bfloat16, 8, 2, 128, 16, 5
    g = torch.Generator(device=device).manual_seed(8)
    prompt = [33, 1, 16]
    table, N = pages_for(g, [n + steps for n in prompt], page)
    kc, vc = cache_pair(g, N, page, Hk, D, dt, device, "plain")
    inv = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().to(device)
    td = table.to(device)
    lens = torch.zeros(3, dtype=torch.int32, device=device)
    x = torch.randn(sum(prompt), H + 2 * Hk, D, generator=g, device=device).to(dt)
    cu = torch.tensor(np.cumsum([0] + prompt), dtype=torch.int32, device=device)
    paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], kc, vc, td, lens, cu_seqlens=cu, inv_freq=inv)
    lens += torch.tensor(prompt, dtype=torch.int32, device=device)
    for step in range(steps):
        x = torch.randn(3, H + 2 * Hk, D, generator=g, device=device).to(dt)
        q = paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], kc, vc, td, lens, q=x[:, :H],
                            inv_freq=inv)
        lens += 1
        out = paged_decode_attn(q, kc, vc, td, lens)
        ref = op.decode(f64(q), f64(kc), f64(vc), table.numpy(), lens.tolist(), 1 / math.sqrt(D))
        close_decode(out, *ref)


def test_step_under_graph_capture(device):
    """Append and attention of a step in one graph, replayed with other tokens, lengths
    and pages; two graphs of different steps alternate."""
    print("[graph]", flush=True)
    dt, H, Hk, D, page, n = torch.bfloat16, 4, 2, 64, 16, 3
    g = torch.Generator(device=device).manual_seed(9)
    inv = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().to(device)

    def state(k):
        st = {"kc": torch.randn(60, page, Hk, D, generator=g, device=device).to(dt),
              "vc": torch.randn(60, page, Hk, D, generator=g, device=device).to(dt),
              "x": torch.zeros(n, H + 2 * Hk, D, device=device, dtype=dt),
              "table": torch.zeros(n, 20, dtype=torch.int32, device=device),
              "lens": torch.zeros(n, dtype=torch.int32, device=device)}
        refill(st, k)
        return st

    def refill(st, k):
        st["x"].copy_(torch.randn(st["x"].shape, generator=g, device=device).to(dt))
        st["table"].copy_(torch.randperm(60, generator=g, device=device).view(n, 20).int())
        st["lens"].copy_(torch.tensor([(37 * k) % 300, 0, (11 * k + 5) % 19], dtype=torch.int32))

    def step(st):
        x = st["x"]
        q = paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], st["kc"], st["vc"], st["table"],
                            st["lens"], q=x[:, :H], inv_freq=inv)
        return paged_decode_attn(q, st["kc"], st["vc"], st["table"], st["lens"] + 1)

    states = [state(0), state(1)]
    graphs = []
    for st in states:
        step(st)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(st)
        graphs.append((graph, out))
    for k in range(6):
        st, (graph, out) = states[k % 2], graphs[k % 2]
        refill(st, k + 3)
        want = step({**st, "kc": st["kc"].clone(), "vc": st["vc"].clone()})
        torch.cuda.synchronize()
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), k


def test_other_streams(device):
    """Work queued on another stream than the tensors' own."""
    print("[streams]", flush=True)
    lens, q, kc, vc, table, slopes, kw = decode_case(9, device)
    args = (q, kc, vc, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device))
    want = paged_decode_attn(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for s in (side, torch.cuda.current_stream(), side):
        with torch.cuda.stream(s):
            outs.append(paged_decode_attn(*args))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_odd_layouts_are_copied(device):
    """Rows that are not whole 16-byte pieces, and features apart from each other."""
    print("[layouts]", flush=True)
    lens, q, kc, vc, table, slopes, kw = decode_case(0, device)
    args = (kc, vc, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device))
    want = paged_decode_attn(q, *args)
    n, H, D = q.shape
    odd = torch.zeros(n, H, D + 3, device=device, dtype=q.dtype)
    odd[..., :D] = q
    assert torch.equal(paged_decode_attn(odd[..., :D], *args), want)
    assert torch.equal(paged_decode_attn(q.permute(2, 0, 1).contiguous().permute(1, 2, 0), *args),
                       want)
    flat = torch.zeros(q.numel() + 1, device=device, dtype=q.dtype)
    flat[1:] = q.flatten()
    assert torch.equal(paged_decode_attn(flat[1:].view(n, H, D), *args), want)
    # a table that is a part of a wider one, rows of one token
    wide = torch.zeros(n, table.shape[1] + 5, dtype=torch.int32, device=device)
    wide[:, :table.shape[1]] = table.to(device)
    assert torch.equal(paged_decode_attn(q, kc, vc, wide[:, :table.shape[1]], args[3]), want)
    bad = torch.zeros(4, 16, 1, D + 3, device=device, dtype=q.dtype)[..., :D]
    with pytest.raises(ValueError, match="16-byte aligned"):
        paged_decode_attn(q, bad, bad, *args[2:])
    with pytest.raises(ValueError, match="expanded"):
        paged_decode_attn(q, bad[:, :1].contiguous().expand(4, 16, 1, D),
                          bad.contiguous(), *args[2:])


def test_empty_calls(device):
    print("[empty]", flush=True)
    kc = torch.zeros(2, 16, 1, 64, device=device, dtype=torch.bfloat16)
    none = torch.zeros(0, 4, dtype=torch.int32, device=device)
    q = torch.zeros(0, 2, 64, device=device, dtype=torch.bfloat16)
    assert paged_decode_attn(q, kc, kc, none, none[:, 0]).shape == (0, 2, 64)
    out = paged_kv_append(q[:, :1], q[:, :1], kc, kc, none, none[:, 0], q=q)
    assert out.shape == (0, 2, 64)
    # sequences but no tokens
    lens = torch.zeros(3, dtype=torch.int32, device=device)
    cu = torch.zeros(4, dtype=torch.int32, device=device)
    assert paged_kv_append(q[:, :1], q[:, :1], kc, kc, torch.zeros(3, 4, dtype=torch.int32,
                                                                   device=device), lens,
                           cu_seqlens=cu) is None
    # no pages in the table
    out = paged_decode_attn(torch.ones(3, 2, 64, device=device, dtype=torch.bfloat16), kc, kc,
                            torch.zeros(3, 0, dtype=torch.int32, device=device), lens + 5)
    assert not out.any()


def test_caches_past_4_gib(device):
    """Pages beyond 4 GiB of a cache hold and give the same bits as near ones."""
    page, Hk, D, H, dt = 256, 2, 128, 8, torch.bfloat16
    N = (5 << 30) // (page * Hk * D * 2)
    print(f"[far pages] {N} pages", flush=True)
    g = torch.Generator(device=device).manual_seed(12)
    kc = torch.zeros(N, page, Hk, D, device=device, dtype=dt)
    vc = torch.zeros_like(kc)
    x = torch.randn(700, H + 2 * Hk, D, generator=g, device=device).to(dt)
    inv = (10000.0 ** (-torch.arange(0, D, 2) / D)).float().to(device)
    outs = []
    for pages in ([0, 1, 2], [N - 1, N - 3, N - 2]):
        table = torch.tensor([pages], dtype=torch.int32, device=device)
        zero = torch.zeros(1, dtype=torch.int32, device=device)
        q = paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], kc, vc, table, zero,
                            cu_seqlens=torch.tensor([0, 700], dtype=torch.int32, device=device),
                            q=x[:, :H], inv_freq=inv)
        out = paged_decode_attn(q[-1:], kc, vc, table, zero + 700)
        outs.append((q, out, kc[pages].clone(), vc[pages].clone()))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert not kc[3:N - 3].any()
    q, out = outs[0][:2]
    ref = op.decode(f64(q[-1:]), f64(kc[:3]), f64(vc[:3]), np.array([[0, 1, 2]]), [700], D ** -0.5)
    close_decode(out, *ref)


def test_two_threads(device):
    """Decoding from two threads, each on a stream of its own."""
    import threading
    print("[decode threads]", flush=True)
    work, errors = [], []
    for case in (5, 9):
        lens, q, kc, vc, table, slopes, kw = decode_case(case, device)
        args = (q, kc, vc, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device))
        work.append((args, kw, None if slopes is None else slopes.to(device),
                     paged_decode_attn(*args, alibi_slopes=None if slopes is None
                                       else slopes.to(device), **kw)))
    torch.cuda.synchronize()

    def run(args, kw, slopes, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    out = paged_decode_attn(*args, alibi_slopes=slopes, **kw)
                torch.cuda.current_stream().synchronize()
            assert torch.equal(out, want)
        except BaseException as e:
            errors.append(e)
    threads = [threading.Thread(target=run, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_tokens_in_front_of_the_first_sequence(device):
    """cu_seqlens that does not start at 0: the tokens in front belong to no sequence."""
    print("[append cu]", flush=True)
    kc = torch.zeros(2, 16, 1, 64, device=device, dtype=torch.bfloat16)
    vc = torch.zeros_like(kc)
    k = torch.ones(5, 1, 64, device=device, dtype=torch.bfloat16)
    table = torch.tensor([[1]], dtype=torch.int32, device=device)
    q = paged_kv_append(k, k, kc, vc, table, torch.tensor([4], dtype=torch.int32, device=device),
                        cu_seqlens=torch.tensor([3, 5], dtype=torch.int32, device=device), q=k)
    assert not q[:3].any() and q[3:].all()
    want = torch.zeros(16, dtype=torch.bool)
    want[4:6] = True
    assert torch.equal(kc[1, :, 0].any(-1).cpu(), want) and not kc[0].any()


@pytest.mark.parametrize("H,Hk", [(1024, 1), (1024, 1024), (130, 2)])
def test_decode_many_heads(device, H, Hk):
    """Several blocks of 16 heads a key head; as many key heads as there can be."""
    print(f"[decode heads] {H}/{Hk}", flush=True)
    D, page, lens, dt = 64, 16, [700, 0, 33], torch.float16
    g = torch.Generator(device=device).manual_seed(13)
    kc, vc = (torch.randn(50, page, Hk, D, generator=g, device=device).to(dt) for _ in range(2))
    q = torch.randn(3, H, D, generator=g, device=device).to(dt)
    table = torch.arange(3 * 44, dtype=torch.int32).view(3, 44) % 50
    out = paged_decode_attn(q, kc, vc, table.to(device),
                            torch.tensor(lens, dtype=torch.int32, device=device), window=650)
    ref = op.decode(f64(q), f64(kc), f64(vc), table.numpy(), lens, D ** -0.5, window=650)
    close_decode(out, *ref)


def test_expanded_features_are_copied(device):
    """Rows of one repeated feature (stride 0) are laid out before a kernel reads them."""
    print("[expanded]", flush=True)
    lens, q, kc, vc, table, slopes, kw = decode_case(0, device)
    args = (kc, vc, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device))
    n, H, D = q.shape
    wide = torch.randn(n, H, 8, device=device).to(q.dtype)[..., :1].expand(n, H, D)
    assert wide.stride(2) == 0
    assert torch.equal(paged_decode_attn(wide, *args), paged_decode_attn(wide.contiguous(), *args))
    k = wide[:, :1].expand(n, kc.shape[2], D)
    got = paged_kv_append(k, k, kc.clone(), vc.clone(), *args[2:], q=wide)
    assert torch.equal(got, wide)
    k1, v1, k2, v2 = (t.clone() for t in (kc, vc, kc, vc))
    paged_kv_append(k, k, k1, v1, *args[2:])
    paged_kv_append(k.contiguous(), k.contiguous(), k2, v2, *args[2:])
    assert torch.equal(k1, k2) and torch.equal(v1, v2)


def chunks_of(H, kc, table, window):
    """Parts of the tiles' axis in a call, from the workspace of their two pieces each."""
    import ctypes as C

    from varlenabsorbflashattn_amd import _lib
    n_pages, page, Hk, D = kc.shape
    c = _lib.PagedCache(k=1 << 20, v=1 << 20, n_pages=n_pages, page_size=page, Hk=Hk, D=D,
                        k_page=8, k_token=8, k_head=8, v_page=8, v_token=8, v_head=8,
                        page_table=1 << 20, table_stride=table.shape[1],
                        table_width=table.shape[1], cache_lens=1 << 20, n_seq=len(table))
    pairs = Hk * -(-H // Hk // 16)
    size = _lib.lib().vafa_paged_decode_workspace(C.byref(c), H, window or 0)
    return size // (2 * pairs * 16 * (4 * D + 8))


SPLIT = [
    # lens, H, Hk, D, page, softcap, window, dtype; tiles of 128 keys, several in each chunk
    ([20000, 9000, 12345, 3], 48, 8, 128, 32, None, None, torch.float16),
    ([20000, 9000, 12345, 3], 48, 8, 128, 32, None, None, torch.bfloat16),
    ([5000, 800, 16000, 0, 129], 32, 16, 64, 16, None, 6000, torch.bfloat16),
    ([3000, 33, 5000, 1000], 24, 24, 256, 64, 30.0, None, torch.float16),
    ([257, 6000, 1, 2100, 2100], 160, 5, 128, 128, None, None, torch.float16),
]


@pytest.mark.parametrize("case", range(len(SPLIT)))
def test_decode_of_sequences_cut_anywhere(device, case):
    """Chunks that end one sequence and begin the next: a sequence's first piece is then a
    chunk's second partial result.  The bound per element would hide a lost tile of a long
    sequence, so each sequence is held to a 2-norm as well.  There the roundings are
    independent: of P for the product (with |v - o| for |v|, as their sum is the
    denominator) at most u / sqrt(3) in the mean, and of the result as much: 0.82 u."""
    lens, H, Hk, D, page, cap, window, dt = SPLIT[case]
    print(f"[decode cut] {SPLIT[case]}", flush=True)
    g = torch.Generator(device=device).manual_seed(case + 31)
    table, N = pages_for(g, lens, page)
    kc, vc = cache_pair(g, N, page, Hk, D, dt, device, "plain")
    q = torch.randn(len(lens), H, D, generator=g, device=device).to(dt)
    tiles = [-(-min(n, window or n) // 128) for n in lens]
    per = -(-sum(tiles) // chunks_of(H, kc, table, window))
    base = np.cumsum([0] + tiles)
    second = [b for b, n in enumerate(tiles)
              if n and base[b] % per and base[b] // per != (base[b + 1] - 1) // per]
    print(f"  {per} tiles a chunk, sequences from {base[:-1].tolist()}", flush=True)
    assert per >= 2 and second
    kw = {"softcap": cap, "window": window}
    out = paged_decode_attn(q, kc, vc, table.to(device),
                            torch.tensor(lens, dtype=torch.int32, device=device), **kw)
    args = f64(q), f64(kc), f64(vc)
    ref = op.decode(*args, table.numpy(), lens, D ** -0.5, **kw)
    close_decode(out, *ref)
    got, u = f64(out), U[dt]

    def off(x, b):
        return np.linalg.norm(x[b] - ref[0][b]) / np.linalg.norm(ref[0][b]) / u
    for b, n in enumerate(lens):
        if n:
            print(f"  sequence {b}: {off(got, b):.2f} u", flush=True)
            assert off(got, b) < 1.0, b
    # what one tile less would do
    lost = table.numpy().copy()
    for b, n in enumerate(lens):
        at = (n - 1) // 128 // 2 * (128 // page)
        lost[b, at:at + 128 // page] = -1
    short = op.decode(*args, lost, lens, D ** -0.5, **kw)[0]
    for b in second:
        if tiles[b] > 1 and (not window or lens[b] <= window):
            assert off(short, b) > 8.0, b
