"""Cases of the language-model operators: packed attention with masks, scores capped by a
tanh and distance biases; appending to a paged key-value cache with the position rotation;
attention of one new token over that cache.

``own`` chooses between the operators' plain form (elementary torch operations in 32 bits,
whole score matrices of padded batches) and the framework's entry points.

A case is a dict of plain values:

``op``      "packed", "append" or "decode"
``dtype``   "bf16" or "fp16"; ``H`` query heads on ``Hk`` key heads of ``D`` features
``n``       number of sequences, ``lens`` "distribution low high" of their new tokens and
            ``past`` of the tokens in front of them ("uniform 0 0": none)
``lseed``   seed of the drawn lengths: they, and so the work, belong to the case; the order of
            the sequences and all values come from the seed of the inputs

packed: ``mode`` "fwd" or "train" (output and the three gradients), ``window`` keys that a
query sees (0: all), ``cap`` of the scores (0.0: none), ``alibi`` a distance bias,
``prefix`` the share of a sequence's keys that every query may see up to.
append: ``rot`` rotated features, ``inter`` pairs of neighbours, ``page`` tokens of a page.
decode: ``page``, ``window``, ``cap``, ``alibi``; ``lens`` is the whole cache's length.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda:0"


# ---- the cases -----------------------------------------------------------------

def _packed(name, mode, dtype, H, Hk, D, n, lens, past="uniform 0 0", window=0, cap=0.0,
            alibi=False, prefix=0.0, lseed=0):
    return {"name": name, "op": "packed", "mode": mode, "dtype": dtype, "H": H, "Hk": Hk, "D": D,
            "n": n, "lens": lens, "past": past, "window": window, "cap": cap, "alibi": alibi,
            "prefix": prefix, "lseed": lseed}


def _append(name, dtype, H, Hk, D, n, lens, past, page, rot, inter=False, lseed=0):
    return {"name": name, "op": "append", "dtype": dtype, "H": H, "Hk": Hk, "D": D, "n": n,
            "lens": lens, "past": past, "page": page, "rot": rot, "inter": inter, "lseed": lseed}


def _decode(name, dtype, H, Hk, D, n, lens, page, window=0, cap=0.0, alibi=False, lseed=0):
    return {"name": name, "op": "decode", "dtype": dtype, "H": H, "Hk": Hk, "D": D, "n": n,
            "lens": lens, "page": page, "window": window, "cap": cap, "alibi": alibi,
            "lseed": lseed}


def listed():
    return [
        # The prompts of one small request: four short ones, where latency counts.
        _packed("packed_prompt_small", "fwd", "bf16", 16, 4, 64, 4, "log 17 200"),
        # Training on packed documents of long-tailed lengths, causal, grouped key heads.
        _packed("packed_train_causal", "train", "bf16", 16, 4, 128, 16, "log 1 4096"),
        # Training of layers with capped scores and a sliding window, wide heads.
        _packed("packed_train_capped", "train", "fp16", 8, 4, 256, 8, "log 256 4096", window=1024,
                cap=30.0),
        # Training with a distance bias on instructions whose prompt is seen both ways.
        _packed("packed_train_prefix", "train", "bf16", 12, 12, 64, 24, "log 1 1500", alibi=True,
                prefix=0.5),
        # One chunk of each of eight long prompts against what was computed before it.
        _packed("packed_prompt_chunk", "fwd", "bf16", 32, 8, 128, 8, "uniform 100 512",
                past="log 4096 32768"),
        # The cache's side of one decoding step of a small batch.
        _append("append_step_small", "bf16", 32, 8, 128, 8, "uniform 1 1", "log 17 500", 16, 128),
        # The same for a large batch; neighbours rotated, half of the features.
        _append("append_step_batch", "fp16", 16, 16, 64, 256, "uniform 1 1", "log 17 8192", 32, 32,
                inter=True),
        # The prompts of a batch, some behind a prefix that is cached already.
        _append("append_prompt", "bf16", 32, 8, 128, 16, "log 128 8192", "log 1 2048", 64, 128),
        # One decoding step of a small batch with short caches.
        _decode("decode_small", "fp16", 16, 4, 64, 4, "log 17 500", 16),
        # A serving batch with caches of very unequal lengths.
        _decode("decode_batch", "bf16", 32, 8, 128, 64, "log 1024 32768", 16),
        # Two sequences with very long caches, a distance bias.
        _decode("decode_long", "bf16", 32, 4, 128, 2, "log 100000 131071", 256, alibi=True),
        # Layers with capped scores and a sliding window, wide heads.
        _decode("decode_capped", "bf16", 16, 8, 256, 32, "log 500 8192", 64, window=4096,
                cap=50.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    Hk = rng.choice([1, 2, 3, 4, 8])
    return {"H": Hk * rng.choice([1, 2, 4, 5, 8]), "Hk": Hk}


def _scores(rng):
    return {"window": rng.choice([0, 0, _log_int(rng, 16, 2048)]),
            "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "alibi": rng.random() < 0.25}


def _draw_prompt(rng):
    case = _packed("", "fwd", rng.choice(["bf16", "fp16"]), D=rng.choice([64, 128, 128, 256]),
                   n=_log_int(rng, 1, 16), lens=f"log 1 {_log_int(rng, 16, 4096)}", **_heads(rng),
                   **_scores(rng))
    if rng.random() < 0.4:
        case["past"] = f"log 1 {_log_int(rng, 64, 16384)}"
        case["lens"] = f"uniform 1 {_log_int(rng, 1, 512)}"
    return case


def _draw_train(rng):
    case = _packed("", "train", rng.choice(["bf16", "fp16"]), D=rng.choice([64, 128, 128, 256]),
                   n=_log_int(rng, 1, 24), lens=f"log 1 {_log_int(rng, 64, 4096)}", **_heads(rng),
                   **_scores(rng))
    if rng.random() < 0.3:
        case["prefix"] = rng.choice([0.25, 0.5, 1.0])
    return case


def _draw_append(rng):
    D = rng.choice([64, 128, 128, 256])
    step = rng.random() < 0.5
    lens = "uniform 1 1" if step else f"log 1 {_log_int(rng, 16, 8192)}"
    return _append("", rng.choice(["bf16", "fp16"]), D=D,
                   n=_log_int(rng, 1, 256) if step else _log_int(rng, 1, 16), lens=lens,
                   past=f"log 1 {_log_int(rng, 16, 8192)}", page=rng.choice([16, 32, 64, 256]),
                   rot=rng.choice([D, D, D // 2]), inter=rng.random() < 0.3, **_heads(rng))


def _draw_decode(rng):
    return _decode("", rng.choice(["bf16", "fp16"]), D=rng.choice([64, 128, 128, 256]),
                   n=_log_int(rng, 1, 64), lens=f"log 1 {_log_int(rng, 64, 65536)}",
                   page=rng.choice([16, 32, 64, 256]), **_heads(rng), **_scores(rng))


def draw(rng: random.Random):
    """One more case of these ranges: the work, and the plain form's padded score matrix, no
    more than the largest listed case's."""
    most, padded = max(map(_cost, listed())), max(map(_padded, listed()))
    while True:
        case = rng.choice([_draw_prompt, _draw_train, _draw_append, _draw_decode])(rng)
        case["lseed"] = rng.randrange(1 << 16)
        del case["name"]
        if _cost(case) <= most and _padded(case) <= padded:
            return case


# ---- lengths and inputs ----------------------------------------------------------

def _draw_lens(rng, spec, n):
    kind, lo, hi = spec.split()
    lo, hi = int(lo), int(hi)
    if kind == "uniform":
        return rng.integers(lo, hi + 1, size=n)
    x = np.exp(rng.uniform(math.log(lo), math.log(hi), size=n))  # log-uniform
    return np.clip(np.rint(x), lo, hi).astype(np.int64)


def _lens(case, seed=None):
    """(new tokens, tokens in front of them) of each sequence; a seed permutes them."""
    rng = np.random.default_rng(case["lseed"])
    new = _draw_lens(rng, case["lens"], case["n"])
    past = _draw_lens(rng, case.get("past", "uniform 0 0"), case["n"])
    if seed is not None:
        order = np.random.default_rng(seed).permutation(case["n"])
        new, past = new[order], past[order]
    return new, past


def _cu(lens):
    cu = np.zeros(len(lens) + 1, dtype=np.int32)
    cu[1:] = np.cumsum(lens)
    return torch.from_numpy(cu)


def _prefixes(case, nk):
    return np.floor(case["prefix"] * nk).astype(np.int64)


def _slopes(case):
    if not case["alibi"]:
        return None
    H = case["H"]
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=DEVICE)


def _inputs(case, seed):
    """The tensors of one call, on the GPU."""
    new, past = _lens(case, seed)
    H, Hk, D, dt = case["H"], case["Hk"], case["D"], DTYPES[case["dtype"]]
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=dt)

    T = int(new.sum())
    if case["op"] == "packed":
        Tk = int((new + past).sum())
        x = {"q": normal(T, H, D), "k": normal(Tk, Hk, D), "v": normal(Tk, Hk, D)}
        if case["mode"] == "train":
            x["do"] = normal(T, H, D)
        return new, past, x
    # q, k and v are parts of one projection's output
    if case["op"] == "append":
        total, qkv = new + past, normal(T, H + 2 * Hk, D)
        x = {"q": qkv[:, :H], "k": qkv[:, H:H + Hk], "v": qkv[:, H + Hk:]}
    else:
        total = new
        x = {"q": normal(case["n"], H + 2 * Hk, D)[:, :H]}
    pages = -(-total // case["page"])
    N, P = int(pages.sum()) + 3, int(pages.max())
    order = torch.randperm(N, generator=g, device=DEVICE).cpu().numpy().astype(np.int32)
    table, at = np.zeros((case["n"], P), dtype=np.int32), 0
    for b, c in enumerate(pages.tolist()):
        table[b, :c] = order[at:at + c]
        at += c
    x["k_cache"] = normal(N, case["page"], Hk, D)
    x["v_cache"] = normal(N, case["page"], Hk, D)
    x["page_table"] = torch.from_numpy(table).to(DEVICE)
    if case["op"] == "append":
        x["cache_lens"] = torch.from_numpy(past.astype(np.int32)).to(DEVICE)
        x["cu"] = None if T == case["n"] else _cu(new).to(DEVICE)
        R = case["rot"]
        x["inv_freq"] = (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).float().to(
            DEVICE)
    else:
        x["cache_lens"] = torch.from_numpy(total.astype(np.int32)).to(DEVICE)
    return new, past, x


def prepare(case, seed):
    new, past, x = _inputs(case, seed)
    st = {"case": case, "max_new": int(new.max()), "max_len": int((new + past).max()), **x}
    if case["op"] == "packed":
        # lengths come from the data loader, on the host
        st["cu_q"], st["cu_k"] = _cu(new), _cu(new + past)
        st["prefix"] = None
        if case["prefix"]:
            st["prefix"] = torch.from_numpy(_prefixes(case, new + past).astype(np.int32))
    if case["op"] != "append":
        st["slopes"] = _slopes(case)
    return st


def run(st):
    return {"packed": _run_packed, "append": _run_append, "decode": _run_decode}[
        st["case"]["op"]](st)


# ---- packed attention ------------------------------------------------------------

def _run_packed(st):
    case = st["case"]
    if own:
        from varlenabsorbflashattn_amd import packed_masked_attn
        kw = {"cu_seqlens_q": st["cu_q"], "cu_seqlens_k": st["cu_k"], "causal": True,
              "window": case["window"] or None, "softcap": case["cap"] or None,
              "prefix_lens": st["prefix"], "alibi_slopes": st["slopes"]}
        x = [st["q"], st["k"], st["v"]]
        if case["mode"] == "fwd":
            with torch.no_grad():
                return packed_masked_attn(*x, **kw)
        x = [t.detach().requires_grad_(True) for t in x]
        o = packed_masked_attn(*x, **kw)
        return (o.detach(),) + torch.autograd.grad(o, x, st["do"])
    return _plain_packed(case, st)


def _rows(cu, T):
    """(sequence, place in it) of T packed tokens."""
    t = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu[1:], t, right=True)
    return b, t - cu[b]


def _plain_packed(case, st):
    H, Hk, D, n = case["H"], case["Hk"], case["D"], case["n"]
    G, scale = H // Hk, 1.0 / math.sqrt(D)
    cu_q, cu_k = st["cu_q"].to(DEVICE).long(), st["cu_k"].to(DEVICE).long()
    Tq, Tk, Lq, Lk = st["q"].shape[0], st["k"].shape[0], st["max_new"], st["max_len"]
    bq, iq = _rows(cu_q, Tq)
    bk, ik = _rows(cu_k, Tk)
    nq, nk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]

    def pad(x, b, i, L):  # [T, h, D] -> fp32 [n, h, L, D]
        out = torch.zeros((n, x.shape[1], L, D), device=x.device)
        out[b, :, i] = x.float()
        return out

    def group(x):  # [n, H, Lq, D] -> [n * Hk, G * Lq, D]
        return x.reshape(n * Hk, G * Lq, D)

    q = group(pad(st["q"], bq, iq, Lq))
    k = pad(st["k"], bk, ik, Lk).reshape(n * Hk, Lk, D)
    v = pad(st["v"], bk, ik, Lk).reshape(n * Hk, Lk, D)
    j = torch.arange(Lk, device=q.device)
    i = torch.arange(Lq, device=q.device)
    p = (i + (nk - nq)[:, None])[:, :, None]  # [n, Lq, 1]
    seen = j <= p
    if case["window"]:
        seen &= j > p - case["window"]
    if st["prefix"] is not None:
        seen |= j < st["prefix"].to(DEVICE)[:, None, None]
    seen &= (j < nk[:, None, None]) & (i < nq[:, None])[:, :, None]
    seen = seen[:, None, None]  # [n, 1, 1, Lq, Lk]
    wide = (n, Hk, G, Lq, Lk)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).view(wide).mul_(scale)
    th = None
    if case["cap"]:
        th = s.div_(case["cap"]).tanh_()
        s = th * case["cap"]
    if st["slopes"] is not None:
        s -= st["slopes"].view(Hk, G, 1, 1) * (p - j).abs()[:, None, None].float()
    s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = s.sum(-1, keepdim=True)
    s.div_(torch.where(total == 0, torch.ones_like(total), total))
    P = s.view(n * Hk, G * Lq, Lk)
    o = torch.matmul(P, v)

    def rows_q(x):
        return x.view(n, H, Lq, D)[bq, :, iq].to(st["q"].dtype)

    def rows_k(x):
        return x.view(n, Hk, Lk, D)[bk, :, ik].to(st["q"].dtype)

    if case["mode"] == "fwd":
        return rows_q(o)
    do = group(pad(st["do"], bq, iq, Lq))
    dv = torch.matmul(P.transpose(1, 2).contiguous(), do)
    ds = torch.matmul(do, v.transpose(1, 2).contiguous())
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(P).mul_(scale)
    if th is not None:
        ds.mul_(1 - th.view(P.shape).square_())
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(1, 2).contiguous(), q)
    return rows_q(o), rows_q(dq), rows_k(dk), rows_k(dv)


# ---- the cache -------------------------------------------------------------------

def _run_append(st):
    case = st["case"]
    if own:
        from varlenabsorbflashattn_amd import paged_kv_append
        q = paged_kv_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["page_table"],
                            st["cache_lens"], cu_seqlens=st["cu"], q=st["q"],
                            inv_freq=st["inv_freq"], interleaved=case["inter"])
        return q, st["k_cache"], st["v_cache"]
    T, R, page = st["k"].shape[0], case["rot"], case["page"]
    if st["cu"] is None:
        b, pos = torch.arange(T, device=DEVICE), st["cache_lens"].long()
    else:
        b, i = _rows(st["cu"].long(), T)
        pos = st["cache_lens"].long()[b] + i
    angle = pos.double()[:, None, None] * st["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    half = slice(0, R, 2) if case["inter"] else slice(0, R // 2)
    other = slice(1, R, 2) if case["inter"] else slice(R // 2, R)

    def turn(x):
        x = x.float()
        a, c = x[..., half].clone(), x[..., other].clone()
        x[..., half], x[..., other] = a * cos - c * sin, c * cos + a * sin
        return x.to(st["k"].dtype)

    at = st["page_table"].long()[b, pos // page], pos % page
    st["k_cache"][at] = turn(st["k"])
    st["v_cache"][at] = st["v"]
    return turn(st["q"]), st["k_cache"], st["v_cache"]


def _run_decode(st):
    case = st["case"]
    if own:
        from varlenabsorbflashattn_amd import paged_decode_attn
        return paged_decode_attn(st["q"], st["k_cache"], st["v_cache"], st["page_table"],
                                 st["cache_lens"], window=case["window"] or None,
                                 softcap=case["cap"] or None, alibi_slopes=st["slopes"])
    n, H, Hk, D, L = case["n"], case["H"], case["Hk"], case["D"], st["max_len"]
    G, page, scale = H // Hk, case["page"], 1.0 / math.sqrt(D)
    j = torch.arange(L, device=DEVICE)
    at = st["page_table"].long()[:, j // page], (j % page).expand(n, L)
    k = st["k_cache"][at].float().transpose(1, 2).contiguous()  # [n, Hk, L, D]
    v = st["v_cache"][at].float().transpose(1, 2).contiguous()
    lens = st["cache_lens"].long()[:, None]
    seen = j < lens
    if case["window"]:
        seen &= j >= lens - case["window"]
    q = st["q"].float().reshape(n * Hk, G, D)
    s = torch.matmul(q, k.view(n * Hk, L, D).transpose(1, 2).contiguous()).view(n, Hk, G, L)
    s = s * scale
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    if st["slopes"] is not None:
        s = s - st["slopes"].view(Hk, G, 1) * (lens - 1 - j).float()[:, None, None]
    seen = seen[:, None, None]
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    e = e / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(e.view(n * Hk, G, L), v.view(n * Hk, L, D))
    return o.view(n, H, D).to(st["q"].dtype)


# ---- work ------------------------------------------------------------------------

def _pairs(case):
    """Visible (query, key) pairs of one head, over all sequences."""
    new, past = _lens(case)
    if case["op"] == "decode":
        return int(np.minimum(new, case["window"]).sum() if case["window"] else new.sum())
    total = 0
    for nq, nk, pre in zip(new, new + past, _prefixes(case, new + past)):
        p = np.arange(nk - nq, nk)  # positions of the queries
        first = np.maximum(p + 1 - case["window"], 0) if case["window"] else np.zeros_like(p)
        # [first, p] and [0, pre)
        own_keys = p + 1 - first
        total += int((own_keys + np.maximum(np.minimum(pre, first), 0)
                      + np.maximum(pre - (p + 1), 0)).sum())
    return total


def work(case):
    """Each input read once, each output written once; two products per visible (query, key)
    pair forward and five backward; three multiply-adds for each rotated feature."""
    new, past = _lens(case)
    T, H, Hk, D, e = int(new.sum()), case["H"], case["Hk"], case["D"], 2
    if case["op"] == "packed":
        train, Tk = case["mode"] == "train", int((new + past).sum())
        return {"bytes": e * D * (4 if train else 2) * (H * T + Hk * Tk),
                "flops": (14 if train else 4) * H * D * _pairs(case)}
    if case["op"] == "append":
        return {"bytes": e * D * T * (2 * H + 4 * Hk) + 8 * T, "flops": 3 * T * (H + Hk) * case["rot"]}
    seen = _pairs(case)
    return {"bytes": e * D * (2 * Hk * seen + 2 * H * case["n"]) + 4 * (seen // case["page"]),
            "flops": 4 * H * D * seen}


def _cost(case):
    """Seconds at 5 TB/s and 500 TFLOP/s."""
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 5e14)


def _padded(case):
    """Elements of the plain form's score matrix and fp32 copies of the keys."""
    new, past = _lens(case)
    if case["op"] == "append":
        return 0
    L, n = int((new + past).max()), case["n"]
    rows = int(new.max()) if case["op"] == "packed" else 1
    return n * L * (case["H"] * rows + 2 * case["Hk"] * case["D"])


# ---- 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    """What run() returns, in 64 bits: sequence by sequence and head by head."""
    new, past, x = _inputs(case, seed)
    with torch.no_grad():
        return {"packed": _exact_packed, "append": _exact_append, "decode": _exact_decode}[
            case["op"]](case, new, past, x)


def _exact_head(case, q, k, i0, prefix, slope):
    """(P, d score / d product) of one head: q [a, D] at positions i0.., k [b, D]."""
    z = (q @ k.t()) / math.sqrt(case["D"])
    grad = torch.full_like(z, 1 / math.sqrt(case["D"]))
    if case["cap"]:
        t = torch.tanh(z / case["cap"])
        z, grad = case["cap"] * t, grad * (1 - t * t)
    pos = torch.arange(i0, i0 + q.shape[0], device=q.device)[:, None]
    key = torch.arange(k.shape[0], device=q.device)[None, :]
    if slope is not None:
        z = z - slope * (pos - key).abs()
    hidden = key > pos
    if case["window"]:
        hidden |= pos - key >= case["window"]
    hidden &= key >= prefix
    z = torch.where(hidden, torch.full_like(z, -math.inf), z)
    return torch.softmax(z, dim=1), grad  # every query of these cases sees a key


def _exact_packed(case, new, past, x):
    D, G = case["D"], case["H"] // case["Hk"]
    q, k, v, do = x["q"], x["k"], x["v"], x.get("do")
    outs = [torch.zeros(t.shape, dtype=torch.float64, device=t.device)
            for t in ([q] if do is None else [q, q, k, v])]
    slopes = _slopes(case)
    slopes = None if slopes is None else slopes.double().tolist()
    q0 = k0 = 0
    for nq, nk, pre in zip(new.tolist(), (new + past).tolist(),
                           _prefixes(case, new + past).tolist()):
        sq, sk = slice(q0, q0 + nq), slice(k0, k0 + nk)
        q0, k0 = q0 + nq, k0 + nk
        for h in range(case["H"]):
            qh, kh, vh = q[sq, h].double(), k[sk, h // G].double(), v[sk, h // G].double()
            P, grad = _exact_head(case, qh, kh, nk - nq, pre, slopes and slopes[h])
            o = P @ vh
            outs[0][sq, h] = o
            if do is None:
                continue
            g = do[sq, h].double()
            dz = P * (g @ vh.t() - (g * o).sum(1, keepdim=True)) * grad
            outs[1][sq, h] = dz @ kh
            outs[2][sk, h // G] += dz.t() @ qh
            outs[3][sk, h // G] += P.t() @ g
    return outs[0] if do is None else tuple(outs)


def _exact_append(case, new, past, x):
    R, page = case["rot"], case["page"]
    cache = [x["k_cache"].double(), x["v_cache"].double()]
    q64 = x["q"].double()
    t0 = 0
    for b, (a, p) in enumerate(zip(new.tolist(), past.tolist())):
        s = slice(t0, t0 + a)
        t0 += a
        pos = torch.arange(p, p + a, device=q64.device)
        angle = pos.double()[:, None, None] * x["inv_freq"].double()
        unit = torch.polar(torch.ones_like(angle), angle)

        def turn(y):
            y = y.double().clone()
            r = y[..., :R]
            r = r.unflatten(-1, (R // 2, 2)) if case["inter"] else \
                r.unflatten(-1, (2, R // 2)).transpose(-1, -2)
            r = torch.view_as_real(torch.view_as_complex(r.contiguous()) * unit)
            y[..., :R] = (r if case["inter"] else r.transpose(-1, -2)).flatten(-2)
            return y

        rows = x["page_table"][b].long()[pos // page] * page + pos % page
        cache[0].flatten(0, 1)[rows] = turn(x["k"][s])
        cache[1].flatten(0, 1)[rows] = x["v"][s].double()
        q64[s] = turn(x["q"][s])
    return q64, cache[0], cache[1]


def _exact_decode(case, new, past, x):
    n, H, G, page = case["n"], case["H"], case["H"] // case["Hk"], case["page"]
    out = torch.zeros((n, H, case["D"]), dtype=torch.float64, device=DEVICE)
    slopes = _slopes(case)
    for b, length in enumerate(new.tolist()):
        rows = x["page_table"][b, :-(-length // page)].long()
        k, v = (x[c][rows].flatten(0, 1)[:length].double() for c in ("k_cache", "v_cache"))
        for hk in range(case["Hk"]):
            hs = slice(hk * G, (hk + 1) * G)
            q = x["q"][b, hs].double()
            z = (q @ k[:, hk].t()) / math.sqrt(case["D"])
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            back = torch.arange(length - 1, -1, -1, device=DEVICE)
            if slopes is not None:
                z = z - slopes[hs].double()[:, None] * back
            if case["window"]:
                z[:, back >= case["window"]] = -math.inf
            out[b, hs] = torch.softmax(z, dim=1) @ v[:, hk]
    return out
