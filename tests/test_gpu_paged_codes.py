"""Attention over a paged cache of 8-bit codes on the GPU against the 64-bit oracle.

Codes times their power of two are exact in bf16 (and in fp16 at the powers here), so the
bounds are those of 16-bit caches (test_gpu_paged.py) on the values that the codes stand for,
and one more: the random codes here reach scores hundreds apart, so that probabilities fall below
2^-126 and out of fp32, where the power of two gives 0.  Each of at most 2^15 keys then lacks at
most 2^-126 of a value of at most 448 * 2^6 < 2^15: 2^-96 in all.
"""
import math

import numpy as np
import pytest
import torch

from oracle import paged as op
from test_gpu_head_rows import E4M3, E8M0, code_caches, freqs, values
from test_gpu_paged import A, U, f64, pages_for, within
from varlenabsorbflashattn_amd import paged_decode_attn, paged_kv_append

pytestmark = pytest.mark.gpu


def close_decode(out, ref, mag, flat):
    u, a = U[out.dtype], A[out.dtype]
    within("out", out, ref, (2 * u + 2.0 ** -12) * mag + 2 * a * flat + u * np.abs(ref) + a
           + 2.0 ** -96)


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


def decode_case(case, device):
    lens, H, Hk, D, page, cap, window, alibi, dt, layout = DECODE[case]
    g = torch.Generator(device=device).manual_seed(case + 71)
    table, N = pages_for(g, lens, page)
    kc, vc, ks, vs = code_caches(g, N, page, Hk, D, device, layout)
    # codes are spread over e4m3's range: scores of up to hundreds from q of 2^-5
    q = (torch.randn(len(lens), H + 3, D, generator=g, device=device) / 32).to(dt)[:, :H]
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / H) for h in range(H)]) if alibi else None
    return lens, q, kc, vc, ks, vs, table, slopes, {"softcap": cap, "window": window}


@pytest.mark.parametrize("case", range(len(DECODE)))
def test_decode_codes(device, case):
    print(f"[decode codes] {DECODE[case][1:]}", flush=True)
    lens, q, kc, vc, ks, vs, table, slopes, kw = decode_case(case, device)
    out = paged_decode_attn(q, kc, vc, table.to(device),
                            torch.tensor(lens, dtype=torch.int32, device=device),
                            alibi_slopes=None if slopes is None else slopes.to(device),
                            k_scale=ks, v_scale=vs, **kw)
    ref = op.decode(f64(q), values(kc, ks), values(vc, vs), table.numpy(), lens,
                    1 / math.sqrt(q.shape[-1]), slopes=f64(slopes), **kw)
    close_decode(out, *ref)


def test_decode_codes_equal_16_bits(device):
    """The same values in a 16-bit cache give the same bits."""
    for case in (0, 2, 9):
        lens, q, kc, vc, ks, vs, table, slopes, kw = decode_case(case, device)
        args = (table.to(device), torch.tensor(lens, dtype=torch.int32, device=device))
        wide = [torch.from_numpy(values(c, s)).to(device, q.dtype) for c, s in ((kc, ks), (vc, vs))]
        got = paged_decode_attn(q, kc, vc, *args, k_scale=ks, v_scale=vs, **kw)
        assert torch.equal(got, paged_decode_attn(q, *wide, *args, **kw)), case


def test_decode_absent_codes(device):
    """NaN codes and powers of two of absent keys do not reach the result."""
    print("[decode absent codes]", flush=True)
    dt, page, Hk, D, H = torch.bfloat16, 16, 2, 64, 4
    g = torch.Generator(device=device).manual_seed(5)
    lens, window = [37, 90, 200, 5], 50
    table, N = pages_for(g, lens, page, width=13)
    table[1, 4] = N + 3
    table[2, 10], table[2, 11] = -7, 2 ** 31 - 1
    table[3, 0] = -1  # no page at all: zeros
    kc, vc, ks, vs = code_caches(g, N, page, Hk, D, device, "plain")
    seen = torch.zeros(N, page, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(max(0, n - window), n):
            at = op.place(table.numpy(), N, page, b, j)
            if at is not None:
                seen[at] = True
    hidden = (~seen).to(device)
    bad = [t.view(torch.uint8).clone() for t in (kc, vc, ks, vs)]
    for t, value in zip(bad, (127, 255, 255, 255)):
        t[hidden] = value
    q = (torch.randn(4, H, D, generator=g, device=device) / 32).to(dt)
    args = (table.to(device), torch.tensor(lens, dtype=torch.int32, device=device))
    out = paged_decode_attn(q, bad[0].view(E4M3), bad[1].view(E4M3), *args, window=window,
                            k_scale=bad[2].view(E8M0), v_scale=bad[3].view(E8M0))
    ref = op.decode(f64(q), values(kc, ks), values(vc, vs), table.numpy(), lens, 1 / math.sqrt(D),
                    window=window)
    close_decode(out, *ref)
    assert not out[3].any()


def test_steps_on_codes(device):
    """A prompt stored at once, then tokens one at a time, each attended, in a graph too."""
    print("[steps on codes]", flush=True)
    dt, H, Hk, D, page, steps = torch.bfloat16, 8, 2, 128, 16, 5
    g = torch.Generator(device=device).manual_seed(8)
    prompt = [33, 1, 16]
    table, N = pages_for(g, [n + steps for n in prompt], page)
    kc, vc, ks, vs = code_caches(g, N, page, Hk, D, device, "plain")
    sc = {"k_scale": ks, "v_scale": vs}
    w = 1 + 0.1 * torch.randn(2, D, generator=g, device=device)
    kw = {"inv_freq": freqs(D).to(device), "q_weight": w[0], "k_weight": w[1], **sc}
    td = table.to(device)
    lens = torch.zeros(3, dtype=torch.int32, device=device)
    x = torch.randn(sum(prompt), H + 2 * Hk, D, generator=g, device=device).to(dt)
    cu = torch.tensor(np.cumsum([0] + prompt), dtype=torch.int32, device=device)
    paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], kc, vc, td, lens, cu_seqlens=cu, q=x[:, :H], **kw)
    lens += torch.tensor(prompt, dtype=torch.int32, device=device)
    x = torch.empty(3, H + 2 * Hk, D, device=device, dtype=dt)

    def step():
        q = paged_kv_append(x[:, H:H + Hk], x[:, H + Hk:], kc, vc, td, lens, q=x[:, :H], **kw)
        return q, paged_decode_attn(q, kc, vc, td, lens + 1, **sc)

    def check(q, out):
        ref = op.decode(f64(q), values(kc, ks), values(vc, vs), table.numpy(),
                        (lens + 1).tolist(), 1 / math.sqrt(D))
        close_decode(out, *ref)
    x.normal_(generator=g)
    check(*step())
    lens += 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out = step()
    for _ in range(steps - 1):
        x.normal_(generator=g)
        graph.replay()
        check(q, out)
        lens += 1
