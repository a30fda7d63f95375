"""Attention of several new tokens per sequence over a paged cache on the GPU against the
64-bit oracle.  Bounds as in test_gpu_paged.py (probabilities are rounded for the product,
sums take the rounded values), for codes as in test_gpu_paged_codes.py.
"""
import ctypes as C
import math
import threading

import numpy as np
import pytest
import torch

from oracle import paged as op
from test_gpu_head_rows import E4M3, E8M0, code_caches, freqs, values
from test_gpu_paged import U, cache_pair, f64, pages_for
from test_gpu_paged_codes import close_decode
from varlenabsorbflashattn_amd import (_lib, packed_masked_attn, packed_qk_norm_rope,
                                       paged_chunk_attn, paged_decode_attn, paged_kv_append,
                                       paged_kv_gather)

pytestmark = pytest.mark.gpu

CHUNK = [
    # new tokens, cache lens (new ones among them), H, Hk, D, page, cap, window, slopes, codes,
    # dtype, layout
    ([1], [1], 1, 1, 64, 16, None, None, False, False, torch.bfloat16, "plain"),
    ([3, 1, 0, 9], [5, 200, 7, 9], 4, 1, 64, 16, None, None, False, False, torch.bfloat16, "plain"),
    ([64, 65, 130], [64, 300, 131], 8, 8, 128, 16, None, None, False, False, torch.float16,
     "joint"),
    ([33, 2], [1000, 31], 10, 2, 128, 7, None, None, True, False, torch.bfloat16, "heads"),
    ([40, 5, 64], [700, 5, 64], 6, 2, 256, 64, 30.0, None, False, False, torch.float16, "plain"),
    ([70, 100, 1], [900, 100, 1], 4, 4, 64, 1, 5.0, 100, True, False, torch.bfloat16, "plain"),
    ([30, 200], [300, 700], 16, 1, 256, 256, 50.0, 128, False, False, torch.bfloat16, "joint"),
    ([2] * 70 + [90], [40] * 70 + [300], 2, 2, 64, 16, None, None, False, False, torch.bfloat16,
     "plain"),
    ([5], [5000], 3, 1, 128, 48, None, 1, False, False, torch.float16, "plain"),
    ([3, 0, 1], [0, 0, 0], 4, 2, 64, 16, None, None, False, False, torch.bfloat16, "plain"),
    ([9, 200, 4], [4, 130, 2], 4, 2, 64, 16, None, None, False, False, torch.bfloat16, "plain"),
    ([8, 3, 1], [20000, 3, 9000], 8, 4, 128, 32, None, None, False, False, torch.bfloat16, "plain"),
    ([6], [6000], 64, 1, 256, 128, None, 4097, True, False, torch.float16, "heads"),
    ([3, 1, 0, 9], [5, 200, 7, 9], 4, 1, 64, 16, None, None, False, True, torch.bfloat16, "plain"),
    ([64, 65, 13], [64, 300, 131], 8, 8, 128, 16, None, None, False, True, torch.float16, "joint"),
    ([33, 2], [1000, 31], 10, 2, 128, 7, None, 60, True, True, torch.bfloat16, "heads"),
    ([40, 5, 64], [700, 5, 64], 6, 2, 256, 64, 30.0, None, False, True, torch.float16, "plain"),
    ([8, 3, 1], [9000, 3, 4000], 32, 4, 128, 32, None, None, False, True, torch.bfloat16, "plain"),
    ([300], [300], 1, 1, 256, 16, None, 90, False, True, torch.bfloat16, "heads"),
]


def chunk_case(case, device):
    new, lens, H, Hk, D, page, cap, window, alibi, codes, dt, layout = case
    g = torch.Generator(device=device).manual_seed(sum(new) + sum(lens) + H + D)
    table, N = pages_for(g, lens, page)
    kw = {"softcap": cap, "window": window}
    if codes:
        kc, vc, ks, vs = code_caches(g, N, page, Hk, D, device, layout)
        vals, kw = (values(kc, ks), values(vc, vs)), {**kw, "k_scale": ks, "v_scale": vs}
    else:
        kc, vc = cache_pair(g, N, page, Hk, D, dt, device, layout)
        vals = f64(kc), f64(vc)
    # q as a part of a joint projection, with rows of no sequence in front and behind
    T = sum(new) + 5
    q = torch.randn(T, H + 3, D, generator=g, device=device)
    q = (q / 32 if codes else q).to(dt)[:, :H]
    cu = np.cumsum([2] + list(new))
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)]) if alibi else None
    args = (q, kc, vc, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device),
            torch.tensor(cu, dtype=torch.int32, device=device))
    if alibi:
        kw["alibi_slopes"] = slopes.to(device)
    ref = op.chunk(f64(q), *vals, table.numpy(), lens, cu, 1 / math.sqrt(D), cap, window,
                   f64(slopes))
    return args, kw, ref


@pytest.mark.parametrize("case", range(len(CHUNK)))
def test_chunk(device, case):
    print(f"[chunk] {CHUNK[case]}", flush=True)
    args, kw, ref = chunk_case(CHUNK[case], device)
    out = paged_chunk_attn(*args, **kw)
    close_decode(out, *ref)
    cu = args[5].tolist()
    assert not out[:cu[0]].any() and not out[cu[-1]:].any()


def test_chunk_of_one_token_is_decode(device):
    """One new token per sequence: the decoding attention's result, within both roundings."""
    print("[chunk of one]", flush=True)
    args, kw, ref = chunk_case(([1] * 5, [1, 700, 64, 0, 3000], 16, 4, 128, 16, None, 500, True,
                                False, torch.bfloat16, "plain"), device)
    q, kc, vc, table, lens, cu = args
    out = paged_chunk_attn(*args, **kw)
    one = paged_decode_attn(q[2:7], kc, vc, table, lens, **kw)
    close_decode(out, *ref)
    close_decode(one, *(r[2:7] for r in ref))


def test_chunk_matches_packed_pass(device):
    """A prompt in three chunks through the cache, normed and rotated on the way, against one
    packed pass over whole sequences; the last chunk also on keys gathered from the cache."""
    print("[chunks against packed]", flush=True)
    dt, H, Hk, D, page = torch.bfloat16, 8, 2, 128, 16
    g = torch.Generator(device=device).manual_seed(21)
    lens, steps = [150, 33, 90], [[70, 1, 64], [79, 30, 0], [1, 2, 26]]
    x = torch.randn(sum(lens), H + 2 * Hk, D, generator=g, device=device).to(dt)
    w = 1 + 0.1 * torch.randn(2, D, generator=g, device=device)
    kw = {"inv_freq": freqs(D).to(device), "q_weight": w[0], "k_weight": w[1]}
    cu = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32)
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).to(device)
    yq, yk = packed_qk_norm_rope(x[:, :H], x[:, H:H + Hk], pos, **kw)
    v = x[:, H + Hk:].contiguous()
    want = packed_masked_attn(yq, yk, v, cu_seqlens_q=cu, cu_seqlens_k=cu, window=60, softcap=20.0)
    table, N = pages_for(g, lens, page)
    table = table.to(device)
    kc, vc = cache_pair(g, N, page, Hk, D, dt, device, "plain")
    clen = torch.zeros(3, dtype=torch.int32, device=device)
    done = [0, 0, 0]
    for new in steps:
        rows = torch.cat([torch.arange(cu[b] + done[b], cu[b] + done[b] + new[b]) for b in range(3)])
        part = x[rows.to(device)]
        cun = torch.tensor(np.cumsum([0] + new), dtype=torch.int32, device=device)
        q = paged_kv_append(part[:, H:H + Hk], part[:, H + Hk:], kc, vc, table, clen, cu_seqlens=cun,
                            q=part[:, :H], **kw)
        clen += torch.tensor(new, dtype=torch.int32, device=device)
        out = paged_chunk_attn(q, kc, vc, table, clen, cun, window=60, softcap=20.0)
        ref, mag, flat = op.chunk(f64(q), f64(kc), f64(vc), table.cpu().numpy(), clen.tolist(),
                                  cun.tolist(), 1 / math.sqrt(D), 20.0, 60)
        close_decode(out, ref, mag, flat)
        close_decode(want[rows.to(device)], ref, mag, flat)
        done = [a + c for a, c in zip(done, new)]
    total = int(cu[-1])
    k, vv = paged_kv_gather(kc, vc, table, cu.to(device), total)
    assert torch.equal(k, yk) and torch.equal(vv, v)
    again = packed_masked_attn(q, k, vv, cu_seqlens_q=cun, cu_seqlens_k=cu, window=60, softcap=20.0)
    close_decode(again, ref, mag, flat)


def test_chunk_absent_keys(device):
    """Infinities and NaN behind a length, in bad pages or in front of every window do not
    reach the result; tokens that see nothing but absent keys get zeros."""
    for codes in (False, True):
        print(f"[chunk absent] codes {codes}", flush=True)
        dt, page, Hk, D, H, window = torch.bfloat16, 16, 2, 64, 4, 50
        g = torch.Generator(device=device).manual_seed(5)
        new, lens = [10, 70, 3, 5], [37, 90, 200, 5]
        table, N = pages_for(g, lens, page, width=40)
        table[1, 4] = N + 3
        table[2, 10], table[2, 11] = -7, 2 ** 31 - 1
        table[3, 0] = -1  # no page at all: zeros
        cu = np.cumsum([0] + new)
        seen = torch.zeros(N, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(max(0, n - new[b] + 1 - window), n):
                at = op.place(table.numpy(), N, page, b, j)
                if at is not None:
                    seen[at] = True
        hidden = (~seen).to(device)
        q = torch.randn(sum(new), H, D, generator=g, device=device)
        args = (table.to(device), torch.tensor(lens, dtype=torch.int32, device=device),
                torch.tensor(cu, dtype=torch.int32, device=device))
        if codes:
            kc, vc, ks, vs = code_caches(g, N, page, Hk, D, device, "plain")
            q = (q / 32).to(dt)
            bad = [t.view(torch.uint8).clone() for t in (kc, vc, ks, vs)]
            for t, value in zip(bad, (127, 255, 255, 255)):
                t[hidden] = value
            out = paged_chunk_attn(q, bad[0].view(E4M3), bad[1].view(E4M3), *args, window=window,
                                   k_scale=bad[2].view(E8M0), v_scale=bad[3].view(E8M0))
            vals = values(kc, ks), values(vc, vs)
        else:
            kc, vc = cache_pair(g, N, page, Hk, D, dt, device, "plain")
            q = q.to(dt)
            odd = torch.tensor([float("nan"), float("inf"), -float("inf")], device=device).to(dt)
            kb, vb = kc.clone(), vc.clone()
            for t in (kb, vb):
                t[hidden] = odd[torch.randint(3, t[hidden].shape, generator=g, device=device)]
            out = paged_chunk_attn(q, kb, vb, *args, window=window)
            vals = f64(kc), f64(vc)
        ref = op.chunk(f64(q), *vals, table.numpy(), lens, cu, 1 / math.sqrt(D), window=window)
        close_decode(out, *ref)
        assert not out[cu[3]:].any()
        if codes:
            continue
        # lengths past the table count as full, negative ones as none
        far = torch.tensor([2 ** 31 - 1, -4, 40 * page + 1, -2 ** 31], dtype=torch.int32)
        table[0, 3:], table[2, 13:] = -1, N
        out = paged_chunk_attn(q, kc, vc, table.to(device), far.to(device), args[2])
        ref = op.chunk(f64(q), *vals, table.numpy(), far.tolist(), cu, 1 / math.sqrt(D))
        close_decode(out, *ref)


def test_chunk_large_scores(device):
    """Scores in the thousands (one-hot rows) and a negative scale."""
    print("[chunk large]", flush=True)
    args, kw, _ = chunk_case(CHUNK[1], device)
    q, kc, vc, table, lens, cu = args
    q = (q.float() * 30).to(q.dtype)
    for scale in (1.0, -0.05):
        out = paged_chunk_attn(q, *args[1:], scale=scale)
        ref, mag, flat = op.chunk(f64(q), f64(kc), f64(vc), table.cpu().numpy(), lens.tolist(),
                                  cu.tolist(), scale)
        # scores of up to 2000 in fp32: off by 64 products of 2^-24 of their size, so P by 2^-7
        d, u = np.abs(f64(out) - ref), U[q.dtype]
        assert (d <= (2 * u + 2.0 ** -7) * mag + u * np.abs(ref)).all()


SPLIT = [
    # new, lens, H, Hk, D, page, cap, window, slopes, codes, dtype, layout: tiles cut anywhere
    ([100, 70, 3], [9000, 70, 4000], 16, 4, 128, 32, None, None, False, False, torch.float16,
     "plain"),
    ([4, 4, 4, 1], [20000, 9000, 300, 3], 8, 2, 64, 16, None, None, False, False, torch.bfloat16,
     "plain"),
    ([40, 200], [5000, 3000], 4, 2, 256, 64, 30.0, 2000, False, False, torch.bfloat16, "plain"),
    ([90, 33], [6000, 3000], 6, 1, 128, 64, None, None, True, True, torch.float16, "plain"),
]


@pytest.mark.parametrize("case", range(len(SPLIT)))
def test_chunk_tiles_cut_anywhere(device, case):
    """Tiles cut between many chunks.  The bound per element would hide a lost unit of a long
    sequence, so each sequence is held to a 2-norm as well: independent roundings of P for the
    product and of the result are at most u / sqrt(3) each in the mean, 0.82 u."""
    print(f"[chunk cut] {SPLIT[case]}", flush=True)
    args, kw, ref = chunk_case(SPLIT[case], device)
    out = paged_chunk_attn(*args, **kw)
    close_decode(out, *ref)
    again = paged_chunk_attn(*args, **kw)
    assert torch.equal(out, again)
    got, u, cu = f64(out), U[out.dtype], args[5].tolist()
    for b in range(len(cu) - 1):
        r = ref[0][cu[b]:cu[b + 1]]
        off = np.linalg.norm(got[cu[b]:cu[b + 1]] - r) / np.linalg.norm(r) / u
        print(f"  sequence {b}: {off:.2f} u", flush=True)
        assert off < 1.0, b


def test_chunk_bad_cu_stays_inside(device):
    """cu_seqlens that decrease or leave the rows write inside the result alone, and lengths
    that are far off end."""
    print("[chunk bad cu]", flush=True)
    dt, H, Hk, D, page = torch.bfloat16, 4, 2, 64, 16
    kc = torch.zeros(8, page, Hk, D, device=device, dtype=dt)
    table = torch.arange(16, dtype=torch.int32, device=device).view(2, 8) % 8
    lens = torch.tensor([100, 100], dtype=torch.int32, device=device)
    q = torch.ones(30, H, D, device=device, dtype=dt)
    for cu in ([0, 50, 20], [25, 5, 30], [-7, 10, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 3]):
        out = paged_chunk_attn(q, kc, kc, table, lens,
                               torch.tensor(cu, dtype=torch.int32, device=device))
        assert out.shape == q.shape
    torch.cuda.synchronize()


def test_chunk_empty_calls(device):
    print("[chunk empty]", flush=True)
    kc = torch.zeros(2, 16, 1, 64, device=device, dtype=torch.bfloat16)
    none = torch.zeros(0, 4, dtype=torch.int32, device=device)
    q = torch.ones(3, 2, 64, device=device, dtype=torch.bfloat16)
    zero = torch.zeros(1, dtype=torch.int32, device=device)
    assert not paged_chunk_attn(q, kc, kc, none, none[:, 0], zero).any()
    assert paged_chunk_attn(q[:0], kc, kc, none, none[:, 0], zero).shape == (0, 2, 64)
    lens = torch.zeros(3, dtype=torch.int32, device=device)
    cu = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=device)
    table = torch.zeros(3, 0, dtype=torch.int32, device=device)  # no pages in the table
    assert not paged_chunk_attn(q, kc, kc, table, lens + 5, cu).any()
    # sequences without new tokens
    assert not paged_chunk_attn(q, kc, kc, torch.zeros(3, 1, dtype=torch.int32, device=device),
                                lens + 5, 0 * cu).any()


def test_chunk_under_graph_capture(device):
    """Append and attention in a graph, replayed with other rows, lengths, cu and pages; two
    graphs alternate."""
    print("[chunk graph]", flush=True)
    dt, H, Hk, D, page, n, T = torch.bfloat16, 4, 2, 64, 16, 3, 200
    g = torch.Generator(device=device).manual_seed(9)
    inv = freqs(D).to(device)

    def refill(st, k):
        new = [[1, 150, 40], [66, 0, 100], [1, 1, 1], [190, 3, 7]][k % 4]
        st["x"].copy_(torch.randn(st["x"].shape, generator=g, device=device))
        st["table"].copy_(torch.randperm(360, generator=g, device=device).view(n, 120))
        st["lens"].copy_(torch.tensor([(137 * k) % 1700, 0, (11 * k + 5) % 19]))
        st["cu"].copy_(torch.tensor(np.cumsum([0] + new)))

    def state(k):
        st = {"kc": torch.randn(360, page, Hk, D, generator=g, device=device).to(dt),
              "vc": torch.randn(360, page, Hk, D, generator=g, device=device).to(dt),
              "x": torch.zeros(T, H + 2 * Hk, D, device=device, dtype=dt),
              "table": torch.zeros(n, 120, dtype=torch.int32, device=device),
              "lens": torch.zeros(n, dtype=torch.int32, device=device),
              "cu": torch.zeros(n + 1, dtype=torch.int32, device=device)}
        refill(st, k)
        return st

    def step(st):
        x = st["x"]
        q = paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], st["kc"], st["vc"], st["table"],
                            st["lens"], cu_seqlens=st["cu"], q=x[:, :H], inv_freq=inv)
        lens = st["lens"] + (st["cu"][1:] - st["cu"][:-1])
        return paged_chunk_attn(q, st["kc"], st["vc"], st["table"], lens, st["cu"])

    states, graphs = [state(0), state(1)], []
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


def test_chunk_streams_and_layouts(device):
    print("[chunk streams]", flush=True)
    args, kw, _ = chunk_case(SPLIT[0], device)
    q = args[0]
    want = paged_chunk_attn(*args, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for s in (side, torch.cuda.current_stream(), side):
        with torch.cuda.stream(s):
            outs.append(paged_chunk_attn(*args, **kw))
    torch.cuda.synchronize()
    T, H, D = q.shape
    odd = torch.zeros(T, H, D + 3, device=device, dtype=q.dtype)
    odd[..., :D] = q
    outs.append(paged_chunk_attn(odd[..., :D], *args[1:], **kw))
    outs.append(paged_chunk_attn(q.permute(2, 0, 1).contiguous().permute(1, 2, 0), *args[1:], **kw))
    for o in outs:
        assert torch.equal(o, want)


@pytest.mark.parametrize("H,Hk", [(1024, 1024), (1024, 1), (768, 2)])
def test_chunk_many_heads(device, H, Hk):
    """As many sets of heads as workgroups and more."""
    print(f"[chunk heads] {H}/{Hk}", flush=True)
    D, page, dt = 64, 16, torch.float16
    g = torch.Generator(device=device).manual_seed(13)
    kc, vc = (torch.randn(50, page, Hk, D, generator=g, device=device).to(dt) for _ in "kv")
    new, lens = [3, 0, 2], [600, 0, 33]
    q = torch.randn(5, H, D, generator=g, device=device).to(dt)
    table = torch.arange(3 * 40, dtype=torch.int32).view(3, 40) % 50
    cu = np.cumsum([0] + new)
    out = paged_chunk_attn(q, kc, vc, table.to(device),
                           torch.tensor(lens, dtype=torch.int32, device=device),
                           torch.tensor(cu, dtype=torch.int32, device=device))
    ref = op.chunk(f64(q), f64(kc), f64(vc), table.numpy(), lens, cu, D ** -0.5)
    close_decode(out, *ref)


def test_chunk_past_4_gib(device):
    """Pages beyond 4 GiB of a cache give the same bits as near ones."""
    page, Hk, D, H, dt = 256, 2, 128, 8, torch.bfloat16
    N = (5 << 30) // (page * Hk * D * 2)
    print(f"[far pages] {N} pages", flush=True)
    g = torch.Generator(device=device).manual_seed(12)
    kc = torch.zeros(N, page, Hk, D, device=device, dtype=dt)
    vc = torch.zeros_like(kc)
    x = torch.randn(700, H + 2 * Hk, D, generator=g, device=device).to(dt)
    cu = torch.tensor([0, 700], dtype=torch.int32, device=device)
    zero = torch.zeros(1, dtype=torch.int32, device=device)
    outs = []
    for pages in ([0, 1, 2], [N - 1, N - 3, N - 2]):
        table = torch.tensor([pages], dtype=torch.int32, device=device)
        paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], kc, vc, table, zero, cu_seqlens=cu)
        outs.append(paged_chunk_attn(x[:, :H], kc, vc, table, zero + 700, cu))
    assert torch.equal(*outs) and outs[0].any()


@pytest.mark.parametrize("seed", range(12))
def test_chunk_random(device, seed):
    """Drawn shapes, a third of them many short pieces of narrow heads (which groups of waves
    share)."""
    rng = np.random.default_rng(seed)
    D = 64 if seed % 3 == 0 else int(rng.choice([64, 128, 256]))
    Hk = int(rng.choice([1, 2, 4]))
    n = int(rng.integers(1, 9))
    new = [int(x) for x in rng.integers(0, 9 if seed % 3 == 0 else 150, n)]
    lens = [x + int(rng.integers(0, 1500)) for x in new]
    codes = bool(rng.integers(0, 2)) and seed % 3 != 0
    case = (new, lens, Hk * int(rng.choice([1, 3, 4, 8])), Hk, D, int(rng.choice([3, 16, 64])),
            30.0 if rng.integers(0, 4) == 0 else None,
            int(rng.integers(1, 600)) if rng.integers(0, 3) == 0 else None,
            bool(rng.integers(0, 4) == 0), codes,
            torch.float16 if rng.integers(0, 2) else torch.bfloat16, "plain")
    print(f"[chunk drawn] {case}", flush=True)
    args, kw, ref = chunk_case(case, device)
    out = paged_chunk_attn(*args, **kw)
    close_decode(out, *ref)
    assert torch.equal(out, paged_chunk_attn(*args, **kw))


def test_threads_with_streams(device):
    """Two threads, each on its own stream: attention over a cache, and norms with their
    backward, give what they give alone."""
    print("[two threads]", flush=True)
    errors, jobs = [], []
    for k, case in enumerate((SPLIT[1], SPLIT[2])):
        args, kw, _ = chunk_case(case, device)
        g = torch.Generator(device=device).manual_seed(k)
        x = torch.randn(700, 6, 64, generator=g, device=device).to(torch.bfloat16)
        pos = torch.arange(700, dtype=torch.int32, device=device)
        w = torch.rand(64, generator=g, device=device) + 0.5

        def job(args=args, kw=kw, x=x, pos=pos, w=w):
            q, k_, wq = (t.detach().clone().requires_grad_() for t in (x[:, :4], x[:, 4:], w))
            yq, yk = packed_qk_norm_rope(q, k_, pos, inv_freq=freqs(64).to(x.device), q_weight=wq,
                                         k_weight=wq)
            grads = torch.autograd.grad((yq.float() * x[:, :4]).sum() + yk.float().sum(),
                                        (q, k_, wq))
            return [paged_chunk_attn(*args, **kw), yq.detach(), yk.detach(), *grads]

        jobs.append((job, job()))
    torch.cuda.synchronize()

    def work(job, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = job()
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


@pytest.mark.parametrize("H,Hk,D,lens,window,cap", [
    (8, 2, 64, [9000, 3000], None, None), (8, 1, 64, [7000, 5000], 3000, 30.0),
    (16, 4, 128, [9000, 4000], None, None), (10, 2, 128, [6000, 5000], None, None),
    (4, 2, 256, [5000, 3000], None, None), (6, 2, 256, [5000, 3000], 2000, 30.0)])
@pytest.mark.parametrize("new", [[70, 33], [4, 1]])
def test_chunk_over_codes_cut_anywhere(device, H, Hk, D, lens, window, cap, new):
    """Ordinary rows stored in 8 bits, which many keys share the softmax of: a unit that a cut
    tile lost would show in the sequence's 2-norm (bound as in test_chunk_tiles_cut_anywhere)."""
    print(f"[chunk codes cut] {H}/{Hk} of {D}, {new} behind {lens}", flush=True)
    dt, page = torch.bfloat16, 64
    g = torch.Generator(device=device).manual_seed(H + D + sum(new))
    table, N = pages_for(g, lens, page)
    kc, vc = (torch.zeros(N, page, Hk, D, device=device).to(E4M3) for _ in "kv")
    ks, vs = (torch.zeros(N, page, Hk, dtype=torch.uint8, device=device).view(E8M0) for _ in "kv")
    kv = torch.randn(sum(lens), 2 * Hk, D, generator=g, device=device).to(dt)
    dev_table = table.to(device)
    cl = torch.tensor(lens, dtype=torch.int32, device=device)
    paged_kv_append(kv[:, :Hk], kv[:, Hk:], kc, vc, dev_table, 0 * cl, k_scale=ks, v_scale=vs,
                    cu_seqlens=torch.tensor(np.cumsum([0] + lens), dtype=torch.int32,
                                            device=device))
    q = torch.randn(sum(new), H, D, generator=g, device=device).to(dt)
    cu = np.cumsum([0] + new)
    out = paged_chunk_attn(q, kc, vc, dev_table, cl,
                           torch.tensor(cu, dtype=torch.int32, device=device), window=window,
                           softcap=cap, k_scale=ks, v_scale=vs)
    ref = op.chunk(f64(q), values(kc, ks), values(vc, vs), table.numpy(), lens, cu,
                   1 / math.sqrt(D), cap, window)
    close_decode(out, *ref)
    got, u = f64(out), U[dt]
    for b in range(len(lens)):
        r = ref[0][cu[b]:cu[b + 1]]
        off = np.linalg.norm(got[cu[b]:cu[b + 1]] - r) / np.linalg.norm(r) / u
        print(f"  sequence {b}: {off:.2f} u", flush=True)
        assert off < 1.0, b


@pytest.mark.parametrize("width", [8, 100])  # whole tiles, and tiles that are cut
@pytest.mark.parametrize("codes", [False, True])
def test_chunk_bad_cu_writes_only_its_rows(device, width, codes):
    """cu_seqlens that decrease or leave the rows: nothing in front of or behind the result and
    the workspace changes, and where the end alone is behind the rows, the sequences in front of
    it have their values."""
    H, Hk, D, page, T, G = 4, 2, 64, 16, 30, 4096
    print(f"[chunk guards] table of {width}, codes {codes}", flush=True)
    g = torch.Generator(device=device).manual_seed(width)
    L = _lib.lib()
    if codes:
        kc, vc, ks, vs = code_caches(g, width, page, Hk, D, device, "plain")
        ref_kv = values(kc, ks), values(vc, vs)
        sc = _lib.RowScales(k=ks.data_ptr(), v=vs.data_ptr(), k_page=page * Hk, k_token=Hk,
                            k_head=1, v_page=page * Hk, v_token=Hk, v_head=1)
    else:
        kc, vc = cache_pair(g, width, page, Hk, D, torch.bfloat16, device, "plain")
        ref_kv, sc = (f64(kc), f64(vc)), None
    q = (torch.randn(T, H, D, generator=g, device=device) / 32).to(torch.bfloat16)
    table = torch.arange(width, dtype=torch.int32, device=device).repeat(2, 1)
    lens = torch.tensor([16 * width - 9, 100], dtype=torch.int32, device=device)
    c = _lib.PagedCache(k=kc.data_ptr(), v=vc.data_ptr(), n_pages=width, page_size=page, Hk=Hk,
                        D=D, k_page=page * Hk * D, k_token=Hk * D, k_head=D,
                        v_page=page * Hk * D, v_token=Hk * D, v_head=D,
                        page_table=table.data_ptr(), table_stride=width, table_width=width,
                        cache_lens=lens.data_ptr(), n_seq=2)
    need = L.vafa_paged_chunk_workspace(C.byref(c), T, H, 0)
    assert (need > 0) == (width > 8)
    far = 2 ** 31 - 1
    for cu in ([3, 20, far], [0, 12, 5], [0, 30, -far], [-7, 10, 10], [25, 5, 30], [far, -far, 3],
               [0, 50, 20], [-9, -3, -20]):
        cu_dev = torch.tensor(cu, dtype=torch.int32, device=device)
        out = torch.full((2 * G + T * H * D,), 7.0, device=device, dtype=torch.bfloat16)
        ws = torch.full((2 * G + need,), 0xA5, device=device, dtype=torch.uint8)
        rc = L.vafa_paged_chunk(C.byref(c), None if sc is None else C.byref(sc), q.data_ptr(),
                                H * D, D, T, H, cu_dev.data_ptr(), out[G:].data_ptr(), 0.125, 0.0,
                                0, None, _lib.DT_BF16, ws[G:].data_ptr() if need else None, need,
                                torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert rc == 0, L.vafa_last_error()
        assert (out[:G] == 7).all() and (out[-G:] == 7).all(), cu
        assert (ws[:G] == 0xA5).all() and (ws[G + need:] == 0xA5).all(), cu
        if cu[2] != far:
            continue
        a, b = cu[0], cu[1]
        ref = op.chunk(f64(q)[a:b], *ref_kv, table.cpu().numpy()[:1], [int(lens[0])], [0, b - a],
                       0.125)
        close_decode(out[G:-G].view(T, H, D)[a:b], *ref)


def test_chunk_bad_rows_stay_in_their_sequence(device):
    """NaN in a row of q stays in that row, and in the newest key and value of a sequence in that
    sequence: the others have the bits that they had."""
    for new, lens in (([3, 40, 5], [900, 64, 33]), ([2, 2, 90], [30, 12, 200])):
        for D, H, Hk in ((64, 8, 2), (128, 6, 2), (256, 4, 4)):
            print(f"[chunk bad rows] {new} {lens} D {D}", flush=True)
            args, kw, _ = chunk_case((new, lens, H, Hk, D, 16, None, None, False, False,
                                      torch.bfloat16, "plain"), device)
            q, kc, vc, table, clen, cu = args
            want = paged_chunk_attn(*args, **kw)
            rows = cu.tolist()
            bad = q.clone()
            bad[rows[1] + 1, 1] = float("nan")
            got = paged_chunk_attn(bad, *args[1:], **kw)
            assert got[rows[1] + 1, 1].isnan().all()
            got[rows[1] + 1, 1] = want[rows[1] + 1, 1]
            assert torch.equal(got, want)
            at = op.place(table.cpu().numpy(), kc.shape[0], 16, 1, lens[1] - 1)
            kb, vb = kc.clone(), vc.clone()
            kb[at], vb[at] = float("nan"), float("inf")
            got = paged_chunk_attn(q, kb, vb, *args[3:], **kw)
            assert got[rows[2] - 1].isnan().all()
            keep = torch.ones(len(q), dtype=torch.bool, device=device)
            keep[rows[1]:rows[2]] = False
            assert torch.equal(got[keep], want[keep])
