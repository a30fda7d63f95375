"""Cases of the paged cache's further operators and of what feeds it: attention of several
new tokens per sequence over the pages, caches held in 8 bits (written, read back, attended
to), and the norms of queries and keys with the position rotation, forward and backward.

``own`` chooses between the operators' plain form (elementary torch operations in 32 bits,
whole score matrices of padded batches) and the framework's entry points.

A case is a dict of plain values:

``op``      "chunk", "decode", "append" or "norm"
``dtype``   "bf16" or "fp16"; ``H`` query heads on ``Hk`` key heads of ``D`` features
``n``       number of sequences, ``lens`` "distribution low high" of their new tokens and
            ``past`` of the tokens in front of them ("uniform 0 0": none)
``lseed``   seed of the drawn lengths: they, and so the work, belong to the case; the order of
            the sequences and all values come from the seed of the inputs
``page``    tokens of a page; ``fp8`` caches of 8-bit codes, a power of two for each row

chunk: ``lens`` new tokens behind ``past``, all in the cache; ``window`` keys that a query sees
(0: all), ``cap`` of the scores (0.0: none), ``alibi`` a distance bias.
decode: one new token, ``lens`` is the whole cache's length; always 8-bit caches.
append: norm, rotation and 8-bit rounding of the new tokens, then the cache read back:
``whole`` from the first token on, or the new ones alone.
norm: ``mode`` "fwd" or "train" (outputs and the four gradients).
append, norm: ``rot`` rotated features, ``inter`` pairs of neighbours, ``weights`` "fp32" or
"same" (the inputs' type).

A row (the D features of one token and key head) in 8 bits: e is the least integer with
max |x| <= 448 * 2^e, and x is held as the e4m3 number nearest to x / 2^e, beside 2^e.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda:0"
EPS = 1e-6


# ---- the cases -----------------------------------------------------------------

def _chunk(name, dtype, H, Hk, D, n, lens, past, page, fp8=False, window=0, cap=0.0, alibi=False,
           lseed=0):
    return {"name": name, "op": "chunk", "dtype": dtype, "H": H, "Hk": Hk, "D": D, "n": n,
            "lens": lens, "past": past, "page": page, "fp8": fp8, "window": window, "cap": cap,
            "alibi": alibi, "lseed": lseed}


def _decode(name, dtype, H, Hk, D, n, lens, page, window=0, cap=0.0, alibi=False, lseed=0):
    return {"name": name, "op": "decode", "dtype": dtype, "H": H, "Hk": Hk, "D": D, "n": n,
            "lens": lens, "page": page, "fp8": True, "window": window, "cap": cap,
            "alibi": alibi, "lseed": lseed}


def _append(name, dtype, H, Hk, D, n, lens, past, page, rot, whole, inter=False, weights="fp32",
            lseed=0):
    return {"name": name, "op": "append", "dtype": dtype, "H": H, "Hk": Hk, "D": D, "n": n,
            "lens": lens, "past": past, "page": page, "fp8": True, "rot": rot, "whole": whole,
            "inter": inter, "weights": weights, "lseed": lseed}


def _norm(name, mode, dtype, H, Hk, D, n, lens, rot, inter=False, weights="fp32", lseed=0):
    return {"name": name, "op": "norm", "mode": mode, "dtype": dtype, "H": H, "Hk": Hk, "D": D,
            "n": n, "lens": lens, "rot": rot, "inter": inter, "weights": weights, "lseed": lseed}


def listed():
    return [
        # A few drafted tokens of each of four short sequences, checked at once.
        _chunk("chunk_draft_small", "bf16", 16, 4, 64, 4, "uniform 2 8", "log 17 500", 16),
        # The same for a serving batch with long caches.
        _chunk("chunk_draft_batch", "bf16", 32, 8, 128, 32, "uniform 1 8", "log 1024 32768", 16),
        # One chunk of each of eight long prompts.
        _chunk("chunk_prompt", "bf16", 32, 8, 128, 8, "uniform 100 512", "log 4096 32768", 64),
        # Short turns of many conversations, 8-bit cache.
        _chunk("chunk_turns_fp8", "bf16", 32, 4, 128, 24, "log 1 512", "log 1 16384", 32, fp8=True),
        # Layers with capped scores and a sliding window, wide heads.
        _chunk("chunk_capped", "fp16", 16, 8, 256, 8, "log 16 512", "log 64 8192", 64, window=2048,
               cap=50.0),
        # One decoding step of a small batch with short 8-bit caches.
        _decode("decode_fp8_small", "fp16", 16, 4, 64, 4, "log 17 500", 16),
        # A serving batch with 8-bit caches of very unequal lengths.
        _decode("decode_fp8_batch", "bf16", 32, 8, 128, 64, "log 1024 32768", 16),
        # Layers with capped scores and a sliding window, wide heads, 8-bit cache.
        _decode("decode_fp8_capped", "bf16", 16, 8, 256, 32, "log 500 8192", 64, window=4096,
                cap=50.0),
        # The cache's side of one decoding step of a large batch, queries and keys normed.
        _append("append_fp8_step", "bf16", 32, 8, 128, 256, "uniform 1 1", "log 17 8192", 32, 128,
                False),
        # The prompts of a batch, some behind a prefix; the whole caches read back.
        _append("append_fp8_prompt", "bf16", 32, 8, 128, 16, "log 128 8192", "log 1 2048", 64, 128,
                True),
        # The prompts of one small request: four short ones, neighbours rotated, half of the
        # features.
        _norm("norm_prompt_small", "fwd", "fp16", 16, 4, 64, 4, "log 17 200", 32, inter=True,
              weights="same"),
        # Training on packed documents of long-tailed lengths.
        _norm("norm_train", "train", "bf16", 32, 8, 128, 16, "log 128 8192", 128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    Hk = rng.choice([1, 2, 3, 4, 8])
    return {"H": Hk * rng.choice([1, 2, 4, 5, 8]), "Hk": Hk}


def _scores(rng):
    return {"window": rng.choice([0, 0, _log_int(rng, 16, 4096)]),
            "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "alibi": rng.random() < 0.25}


def _draw_chunk(rng):
    new = rng.choice([f"uniform 1 {_log_int(rng, 1, 512)}", f"log 1 {_log_int(rng, 2, 1024)}"])
    past = rng.choice(["uniform 0 0"] + 3 * [f"log 1 {_log_int(rng, 16, 32768)}"])
    return _chunk("", rng.choice(["bf16", "fp16"]), D=rng.choice([64, 128, 128, 256]),
                  n=_log_int(rng, 1, 48), lens=new, past=past, page=rng.choice([16, 32, 64, 256]),
                  fp8=rng.random() < 0.5, **_heads(rng), **_scores(rng))


def _draw_decode(rng):
    return _decode("", rng.choice(["bf16", "fp16"]), D=rng.choice([64, 128, 128, 256]),
                   n=_log_int(rng, 1, 64), lens=f"log 1 {_log_int(rng, 64, 65536)}",
                   page=rng.choice([16, 32, 64, 256]), **_heads(rng), **_scores(rng))


def _draw_rot(rng):
    D = rng.choice([64, 128, 128, 256])
    return {"D": D, "rot": rng.choice([D, D, D // 2]), "inter": rng.random() < 0.3,
            "weights": rng.choice(["fp32", "same"])}


def _draw_append(rng):
    step = rng.random() < 0.5
    return _append("", rng.choice(["bf16", "fp16"]),
                   n=_log_int(rng, 1, 256) if step else _log_int(rng, 1, 16),
                   lens="uniform 1 1" if step else f"log 1 {_log_int(rng, 16, 8192)}",
                   past=f"log 1 {_log_int(rng, 16, 8192)}", page=rng.choice([16, 32, 64, 256]),
                   whole=not step, **_draw_rot(rng), **_heads(rng))


def _draw_norm(rng):
    return _norm("", rng.choice(["fwd", "train", "train"]), rng.choice(["bf16", "fp16"]),
                 n=_log_int(rng, 1, 24), lens=f"log 1 {_log_int(rng, 16, 8192)}", **_draw_rot(rng),
                 **_heads(rng))


def draw(rng: random.Random):
    """One more case of these ranges: the work, and the plain form's padded score matrix, no
    more than the largest listed case's."""
    most, padded = max(map(_cost, listed())), max(map(_padded, listed()))
    while True:
        case = rng.choice([_draw_chunk, _draw_chunk, _draw_decode, _draw_append, _draw_norm])(rng)
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


def _ints(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(DEVICE)


def _cu(lens):
    return _ints(np.concatenate(([0], np.cumsum(lens))))


def _slopes(case):
    if not case["alibi"]:
        return None
    H = case["H"]
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device=DEVICE)


def _power(e):
    """2^(e - 127) of integers from 1 to 254, from its bits (a power function rounds)."""
    return (e.int() << 23).view(torch.float32)


def _code_rows(x):
    """Rows of fp32 in 8 bits: (codes, the powers of two's exponents plus 127)."""
    amax = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)  # amax = m 2^e, 0.5 <= m < 1, and 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9).clamp_(min=-126)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    codes = (x * _power(127 - e)).to(torch.float8_e4m3fn)
    return codes, (e.squeeze(-1) + 127).to(torch.uint8)


def _inputs(case, seed):
    """The tensors of one call, on the GPU."""
    new, past = _lens(case, seed)
    H, Hk, D, dt = case["H"], case["Hk"], case["D"], DTYPES[case["dtype"]]
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE, dtype=dt)

    T = int(new.sum())
    x = {}
    if case["op"] in ("append", "norm"):
        # q, k and v are parts of one projection's output
        qkv = normal(T, H + 2 * Hk, D)
        x["q"], x["k"], x["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        for name in ("q_weight", "k_weight"):
            w = 1 + 0.1 * torch.randn(D, generator=g, device=DEVICE)
            x[name] = w if case["weights"] == "fp32" else w.to(dt)
        R = case["rot"]
        x["inv_freq"] = (10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)).float().to(
            DEVICE)
    if case["op"] == "norm":
        x["positions"] = _ints(np.concatenate([np.arange(c) for c in new]))
        if case["mode"] == "train":
            x["dq"], x["dk"] = normal(T, H, D), normal(T, Hk, D)
        return new, past, x
    if case["op"] in ("chunk", "decode"):
        x["q"] = normal(T if case["op"] == "chunk" else case["n"], H + 2 * Hk, D)[:, :H]
    total = new if case["op"] == "decode" else new + past
    pages = -(-total // case["page"])
    N, P = int(pages.sum()) + 3, int(pages.max())
    order = torch.randperm(N, generator=g, device=DEVICE).cpu().numpy().astype(np.int32)
    table, at = np.zeros((case["n"], P), dtype=np.int32), 0
    for b, c in enumerate(pages.tolist()):
        table[b, :c] = order[at:at + c]
        at += c
    for kv in "kv":
        c = normal(N, case["page"], Hk, D)
        if case["fp8"]:
            codes, scale = torch.empty_like(c, dtype=torch.float8_e4m3fn), []
            for i in range(0, N, 4096):
                codes[i:i + 4096], s = _code_rows(c[i:i + 4096].float())
                scale.append(s)
            x[kv + "_cache"] = codes
            x[kv + "_scale"] = torch.cat(scale).view(torch.float8_e8m0fnu)
        else:
            x[kv + "_cache"], x[kv + "_scale"] = c, None
    x["page_table"] = torch.from_numpy(table).to(DEVICE)
    x["cache_lens"] = _ints(past if case["op"] == "append" else total)
    if case["op"] != "decode":
        x["cu"] = _cu(new)
    if case["op"] == "append":  # what is read back: rows of each sequence, from a position on
        x["read_cu"] = _cu(total if case["whole"] else new)
        x["read_from"] = _ints(0 * past if case["whole"] else past)
    return new, past, x


def prepare(case, seed):
    new, past, x = _inputs(case, seed)
    st = {"case": case, "max_new": int(new.max()), "max_len": int((new + past).max()), **x}
    if case["op"] == "append":
        st["read_rows"] = int((new + past).sum()) if case["whole"] else int(new.sum())
    if case["op"] in ("chunk", "decode"):
        st["slopes"] = _slopes(case)
    return st


def run(st):
    return {"chunk": _run_chunk, "decode": _run_decode, "append": _run_append,
            "norm": _run_norm}[st["case"]["op"]](st)


# ---- attention over the cache ----------------------------------------------------

def _kw(st):
    case = st["case"]
    return {"window": case["window"] or None, "softcap": case["cap"] or None,
            "alibi_slopes": st["slopes"], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _run_chunk(st):
    if own:
        from varlenabsorbflashattn_amd import paged_chunk_attn
        return paged_chunk_attn(st["q"], st["k_cache"], st["v_cache"], st["page_table"],
                                st["cache_lens"], st["cu"], **_kw(st))
    return _plain_attn(st, st["cu"].long(), st["max_new"])


def _run_decode(st):
    if own:
        from varlenabsorbflashattn_amd import paged_decode_attn
        return paged_decode_attn(st["q"], st["k_cache"], st["v_cache"], st["page_table"],
                                 st["cache_lens"], **_kw(st))
    return _plain_attn(st, torch.arange(st["case"]["n"] + 1, device=DEVICE), 1)


def _values(st, kv, at):
    """Rows of a cache at (pages, slots), fp32: codes times their power of two."""
    if st[kv + "_scale"] is None:
        return st[kv + "_cache"][at].float()
    x = st[kv + "_cache"].view(torch.uint8)[at].view(torch.float8_e4m3fn).float()
    return x.mul_(_power(st[kv + "_scale"].view(torch.uint8)[at]).unsqueeze(-1))


def _rows(cu, T):
    """(sequence, place in it) of T packed tokens."""
    t = torch.arange(T, device=cu.device)
    b = torch.searchsorted(cu[1:], t, right=True)
    return b, t - cu[b]


def _plain_attn(st, cu, Lq):
    case = st["case"]
    n, H, Hk, D, Lk = case["n"], case["H"], case["Hk"], case["D"], st["max_len"]
    G, page, scale, T = H // Hk, case["page"], 1.0 / math.sqrt(D), st["q"].shape[0]
    j = torch.arange(Lk, device=DEVICE)
    at = st["page_table"].long()[:, j // page], (j % page).expand(n, Lk)
    k = _values(st, "k", at).permute(0, 2, 3, 1).contiguous().view(n * Hk, D, Lk)
    v = _values(st, "v", at).transpose(1, 2).contiguous().view(n * Hk, Lk, D)
    b, i = _rows(cu, T)
    q = torch.zeros((n, H, Lq, D), device=DEVICE)
    q[b, :, i] = st["q"].float()
    lens, new = st["cache_lens"].long()[:, None], (cu[1:] - cu[:-1])[:, None]
    row = torch.arange(Lq, device=DEVICE)
    p = (lens - new + row)[:, :, None]  # positions [n, Lq, 1]
    seen = j <= p
    if case["window"]:
        seen &= j > p - case["window"]
    seen &= (row < new)[:, :, None]
    seen = seen[:, None, None]  # [n, 1, 1, Lq, Lk]
    s = torch.matmul(q.view(n * Hk, G * Lq, D), k).view(n, Hk, G, Lq, Lk).mul_(scale)
    if case["cap"]:
        s = s.div_(case["cap"]).tanh_().mul_(case["cap"])
    if st["slopes"] is not None:
        s -= st["slopes"].view(Hk, G, 1, 1) * (p - j).abs()[:, None, None].float()
    s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = s.sum(-1, keepdim=True)
    s.div_(torch.where(total == 0, torch.ones_like(total), total))
    o = torch.matmul(s.view(n * Hk, G * Lq, Lk), v)
    return o.view(n, H, Lq, D)[b, :, i].to(st["q"].dtype)


# ---- norms, rotation, the cache ----------------------------------------------------

def _turns(pos, inv_freq):
    angle = pos.double()[:, None, None] * inv_freq.double()
    return angle.cos().float(), angle.sin().float()


def _parts(case):
    R = case["rot"]
    if case["inter"]:
        return slice(0, R, 2), slice(1, R, 2)
    return slice(0, R // 2), slice(R // 2, R)


def _normed(x, weight):
    """fp32 (x r w, x r, r) with r = 1 / sqrt(mean of squares + eps)."""
    x = x.float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    u = x * r
    return u * weight.float(), u, r


def _turn(case, y, cos, sin):
    first, second = _parts(case)
    a, c = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * cos - c * sin, c * cos + a * sin
    return y


def _run_append(st):
    case, dt = st["case"], st["k"].dtype
    caches = [st[x] for x in ("k_cache", "v_cache", "page_table")]
    if own:
        from varlenabsorbflashattn_amd import paged_kv_append, paged_kv_gather
        scales = {"k_scale": st["k_scale"], "v_scale": st["v_scale"]}
        q = paged_kv_append(st["k"], st["v"], *caches, st["cache_lens"], cu_seqlens=st["cu"],
                            q=st["q"], inv_freq=st["inv_freq"], interleaved=case["inter"],
                            q_weight=st["q_weight"], k_weight=st["k_weight"], eps=EPS, **scales)
        k, v = paged_kv_gather(*caches, st["read_cu"], st["read_rows"], starts=st["read_from"],
                               dtype=dt, **scales)
        return q, k, v
    page = case["page"]
    table = st["page_table"].long()

    def places(cu, starts, T):
        b, i = _rows(cu.long(), T)
        pos = starts.long()[b] + i
        return pos, (table[b, pos // page], pos % page)

    pos, at = places(st["cu"], st["cache_lens"], st["k"].shape[0])
    cos, sin = _turns(pos, st["inv_freq"])
    q = _turn(case, _normed(st["q"], st["q_weight"])[0], cos, sin).to(dt)
    k = _turn(case, _normed(st["k"], st["k_weight"])[0], cos, sin)
    for kv, x in (("k", k), ("v", st["v"].float())):
        codes, scale = _code_rows(x)
        st[kv + "_cache"].view(torch.uint8)[at] = codes.view(torch.uint8)
        st[kv + "_scale"].view(torch.uint8)[at] = scale
    at = places(st["read_cu"], st["read_from"], st["read_rows"])[1]
    return q, _values(st, "k", at).to(dt), _values(st, "v", at).to(dt)


def _run_norm(st):
    case = st["case"]
    if own:
        from varlenabsorbflashattn_amd import packed_qk_norm_rope
        kw = {"positions": st["positions"], "inv_freq": st["inv_freq"],
              "interleaved": case["inter"], "eps": EPS}
        x = [st[name] for name in ("q", "k", "q_weight", "k_weight")]
        if case["mode"] == "fwd":
            with torch.no_grad():
                return packed_qk_norm_rope(x[0], x[1], q_weight=x[2], k_weight=x[3], **kw)
        x = [t.detach().requires_grad_(True) for t in x]
        q, k = packed_qk_norm_rope(x[0], x[1], q_weight=x[2], k_weight=x[3], **kw)
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), x, (st["dq"], st["dk"]))
    cos, sin = _turns(st["positions"], st["inv_freq"])
    outs, grads, weights = [], [], []
    for name in "qk":
        x, w = st[name], st[name + "_weight"]
        y, u, r = _normed(x, w)
        outs.append(_turn(case, y, cos, sin).to(x.dtype))
        if case["mode"] == "train":
            g = _turn(case, st["d" + name].float(), cos, -sin)  # back by the angle
            weights.append((g * u).sum((0, 1)).to(w.dtype))
            g = g * w.float()
            grads.append((r * (g - u * (g * u).mean(-1, keepdim=True))).to(x.dtype))
    return tuple(outs + grads + weights)


# ---- work ------------------------------------------------------------------------

def _pairs(case):
    """Visible (query, key) pairs of one head, and the keys that some query sees, over all
    sequences."""
    new, past = _lens(case)
    if case["op"] == "decode":
        new, past = np.ones_like(new), new - 1
    pairs = keys = 0
    for nq, nk in zip(new.tolist(), (new + past).tolist()):
        p = np.arange(nk - nq, nk)  # positions of the queries
        first = np.maximum(p + 1 - case["window"], 0) if case["window"] else np.zeros_like(p)
        pairs += int((p + 1 - first).sum())
        keys += nk - int(first[0])
    return pairs, keys


def work(case):
    """Each input read once, each output written once: keys and values that some query sees
    with their powers of two and pages; two products per visible (query, key) pair; six
    operations for each normed feature and three for each rotated one, twice as many backward."""
    new, past = _lens(case)
    T, H, Hk, D, e = int(new.sum()), case["H"], case["Hk"], case["D"], 2
    if case["op"] == "norm":
        train = case["mode"] == "train"
        flops = T * (H + Hk) * (6 * D + 3 * case["rot"])
        return {"bytes": e * D * T * (H + Hk) * (5 if train else 2) + 4 * T,
                "flops": flops * (3 if train else 1)}
    row = D + 1  # of an 8-bit cache
    if case["op"] == "append":
        read = int((new + past).sum()) if case["whole"] else T
        return {"bytes": e * D * T * (2 * H + 2 * Hk) + 2 * Hk * (row * T + (row + e * D) * read)
                + 8 * T, "flops": T * ((H + Hk) * (6 * D + 3 * case["rot"]) + 2 * Hk * 3 * D)}
    pairs, keys = _pairs(case)
    rows = T if case["op"] == "chunk" else case["n"]
    return {"bytes": 2 * Hk * keys * (row if case["fp8"] else e * D) + 2 * e * D * H * rows
            + 4 * (keys // case["page"]), "flops": 4 * H * D * pairs}


def _cost(case):
    """Seconds at 5 TB/s and 500 TFLOP/s."""
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 5e14)


def _padded(case):
    """Elements of the plain form's score matrix and fp32 copies of the keys."""
    if case["op"] in ("append", "norm"):
        return 0
    new, past = _lens(case)
    L, n = int((new + past).max()), case["n"]
    rows = int(new.max()) if case["op"] == "chunk" else 1
    return n * L * (case["H"] * rows + 2 * case["Hk"] * case["D"])


# ---- 64 bits ---------------------------------------------------------------------

def exact(case, seed):
    """What run() returns, in 64 bits: sequence by sequence and head by head."""
    new, past, x = _inputs(case, seed)
    with torch.no_grad():
        return {"chunk": _exact_attn, "decode": _exact_attn, "append": _exact_append,
                "norm": _exact_norm}[case["op"]](case, new, past, x)


def _exact_power(e):
    """2^e of whole numbers, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_cache(x, kv, rows):
    """Rows (indexes over pages and slots) of a cache in 64 bits."""
    cache = x[kv + "_cache"].flatten(0, 1)
    if x[kv + "_scale"] is None:
        return cache[rows].double()
    codes = cache.view(torch.uint8)[rows].view(torch.float8_e4m3fn).double()
    e = x[kv + "_scale"].flatten(0, 1).view(torch.uint8)[rows].long() - 127
    return codes * _exact_power(e)[..., None]


def _exact_attn(case, new, past, x):
    H, G, D, page = case["H"], case["H"] // case["Hk"], case["D"], case["page"]
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device=DEVICE)
    slopes, t0 = _slopes(case), 0
    if case["op"] == "decode":
        new, past = np.ones_like(new), new - 1
    for b, (a, before) in enumerate(zip(new.tolist(), past.tolist())):
        key = torch.arange(before + a, device=DEVICE)
        rows = x["page_table"][b].long()[key // page] * page + key % page
        k, v = _exact_cache(x, "k", rows), _exact_cache(x, "v", rows)
        dist = torch.arange(before, before + a, device=DEVICE)[:, None] - key  # position - key
        hidden = dist < 0
        if case["window"]:
            hidden |= dist >= case["window"]
        for h in range(H):
            z = (x["q"][t0:t0 + a, h].double() @ k[:, h // G].t()) / math.sqrt(D)
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
            if slopes is not None:
                z = z - slopes[h].double() * dist
            z[hidden] = -math.inf  # (every query sees itself)
            out[t0:t0 + a, h] = torch.softmax(z, dim=1) @ v[:, h // G]
        t0 += a
    return out


def _exact_unit(pos, x):
    angle = pos.double()[:, None, None] * x["inv_freq"].double()
    return torch.polar(torch.ones_like(angle), angle)


def _exact_turn(case, y, unit):
    R = case["rot"]
    r = y[..., :R]
    r = r.unflatten(-1, (R // 2, 2)) if case["inter"] else \
        r.unflatten(-1, (2, R // 2)).transpose(-1, -2)
    r = torch.view_as_real(torch.view_as_complex(r.contiguous()) * unit)
    r = (r if case["inter"] else r.transpose(-1, -2)).flatten(-2)
    return torch.cat((r, y[..., R:]), dim=-1)


def _exact_norm_of(x, w):
    return x * w / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)


def _exact_code(x):
    """Rows rounded to 8 bits and back: steps of 2^-3 relative to the power of two below a
    value, of 2^-9 below 2^-6, under the row's own power of two."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 448.0))
    e = torch.where(top > 448.0 * _exact_power(e), e + 1, e)  # (the logarithm's own rounding)
    e = torch.where(top <= 448.0 * _exact_power(e - 1), e - 1, e)
    y = x * _exact_power(-e)
    below = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    below = torch.where(_exact_power(below) > y.abs(), below - 1, below).clamp(min=-6)
    step = _exact_power(below - 3)
    return torch.round(y / step) * step * _exact_power(e)  # (halves go to even)


def _exact_append(case, new, past, x):
    page = case["page"]
    q = torch.empty(x["q"].shape, dtype=torch.float64, device=DEVICE)
    read, t0 = {"k": [], "v": []}, 0
    for b, (a, p) in enumerate(zip(new.tolist(), past.tolist())):
        s = slice(t0, t0 + a)
        t0 += a
        unit = _exact_unit(torch.arange(p, p + a, device=DEVICE), x)
        q[s] = _exact_turn(case, _exact_norm_of(x["q"][s].double(), x["q_weight"].double()), unit)
        k = _exact_turn(case, _exact_norm_of(x["k"][s].double(), x["k_weight"].double()), unit)
        before = torch.arange(p if case["whole"] else 0, device=DEVICE)
        rows = x["page_table"][b].long()[before // page] * page + before % page
        for kv, y in (("k", k), ("v", x["v"][s].double())):
            read[kv] += [_exact_cache(x, kv, rows), _exact_code(y)]
    return q, torch.cat(read["k"]), torch.cat(read["v"])


def _exact_norm(case, new, past, x):
    unit = _exact_unit(x["positions"], x)
    outs, grads, weights = [], [], []
    for name in "qk":
        with torch.enable_grad():
            y = x[name].double().requires_grad_(True)
            w = x[name + "_weight"].double().requires_grad_(True)
            z = _exact_turn(case, _exact_norm_of(y, w), unit)
            if case["mode"] == "train":
                dy, dw = torch.autograd.grad(z, (y, w), x["d" + name].double())
                grads.append(dy)
                weights.append(dw)
        outs.append(z.detach())
    return tuple(outs + grads + weights)
